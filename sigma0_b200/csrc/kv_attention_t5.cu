// Attention of many rows (17 and more new tokens x query heads of a key head) over a 16-bit key / value
// cache: both products on tcgen05, for heads of up to 64 or exactly up to 128 channels with 16-byte
// aligned rows.  The operator is described in kv_attention.cu, the split over CTAs in kv_attention.cuh.
//
// The products are transposed, so that the instruction's 128 rows are keys, then channels, and its 64
// columns the queries (64 rows of a unit; more are further row blocks of it):
//   S^T [128 keys, 64]     = K [128, HD] Q^T        A: K (K-major), B: Q (K-major)
//   O^T [HD channels, 64] += V^T [HD, 128] P^T      A: V read MN-major, B: P^T read MN-major
// Both operands of both products lie in shared memory as they come (128-byte rows, 128-byte swizzle);
// S^T (two buffers) and O^T are in tensor memory, where a softmax thread owns one key and 32 of its scores.
//
// Roles of a CTA (one per SM): warps 0-7 softmax and the unit's output; warp 8 issues the
// products, S of tile i + 1 before O of tile i; warp 11 stores the new rows and turns their mask into bits,
// which takes several trips to a busy memory and nobody waits for; warps 9 and 10 load: K and V tiles go through a ring of slots by
// cp.async (rows past the end become 0, any strides), as far ahead as there are free slots.  Mbarriers
// connect them; every wait is bounded: one that runs out ends all roles, makes the CTA's rows NaN and sets a status word.
//
// A unit costs some 8 tiles besides its own, and 20 at least (kv_attention.cuh has the sweep): the trips for queries, mask
// bits and new rows take 3 us each while the memory is busy, and only the tiles of a long unit cover them.
//
// The softmax's reference moves only when a score passes it by far (see kv_attention_tc.cu); then
// the rows' output in tensor memory is rescaled.  p is rounded once to the cache's type for the second product: a second
// tile for what that leaves does not fit beside the ring at 128 channels, and the error is 1.1 times that of the
// output's own rounding (tree of 64 over 22,000 tokens).  What bounds it: HBM up to 64 rows, if 64 columns x 128
// keys take less than the 64 KB of their K and V take from HBM (2,800 cycles of an SM at the copy rate):
// the products read 6 KB of operands per 16-channel step from shared memory, some 770 cycles a tile; the
// exponentials are 512 cycles of the SM's special function units.  Measured: 2,650-2,800 cycles a tile in a long unit;
// 64 nodes over 16 contexts of up to 22,000 tokens, 16 heads of 128: 379 us with the join, 75% of the copy rate (500 us
// for an mma.sync kernel with 64 rows, whose warps wait for one another's latencies at 44% of that pipe).
#include <algorithm>

#include "kv_attention.cuh"
#include "tc_common.cuh"

namespace s0 {
namespace kv {
namespace t5 {

constexpr int KT = 128, N = 64, PANEL = KT * 128;     // keys of a tile, rows of a unit, bytes of 64 channels of a tile
constexpr int ST = 256, LT = 64, NT = ST + 32 + LT + 32;   // softmax threads, loading threads, threads
constexpr int TM_O = 2 * N, TM_COLS = 256;            // tensor memory: S^T buffers at 0 and N, O^T
constexpr unsigned long long DRAIN_NS = 2000000000ull;  // the bound of the wait for the last products, whatever the others' is
__device__ int gave_up;                               // 1 once a wait has run out on this device
constexpr float UNSET = -3.402823466e38f;                       // the reference of a row that has seen nothing

template <int HD> struct Ring {
  static constexpr int SLOT = HD / 64 * PANEL, SLOTS = HD == 128 ? 5 : 8;
};

struct Bars {
  uint64_t full[8], empty[8], sfull[2], sempty[2], qempty[2], pfull, pdone, mfull[2], mempty[2], drain;
  uint32_t tslot;
  int abort, bad[2];                                  // a wait ran out; a tile of new V is not finite
};
template <int HD> struct Smem {
  static constexpr int Q = Ring<HD>::SLOT * Ring<HD>::SLOTS, QB = N * 128 * (HD / 64), P = Q + 2 * QB, F = P + PANEL;
  static constexpr int BYTES = F + (2 * N + 4 * N + 4 * KT) * 4 + (int)sizeof(Bars) + 1024;   // reference, factor, sums of 4 warps; mask bits
};

// false: the wait took longer than `limit` ns, or another one has
S0_DEV bool wait(uint64_t* bar, uint32_t parity, volatile int* abort, unsigned long long limit) {
  unsigned long long since = 0, now;
  for (int i = 1; limit; ++i) {
    if (tc::mbar_wait(bar, parity, 1)) return true;
    if (*abort) return false;
    if (i & 63) continue;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(now));
    if (since == 0) since = now;
    if (now - since > limit) break;
  }
  *abort = 1;
  return false;
}
// barrier of the softmax threads with a vote
S0_DEV bool any_of(bool x) {
  uint32_t y;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, 1, 256, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}\n"
      : "=r"(y)
      : "r"((uint32_t)x)
      : "memory");
  return y != 0;
}
S0_DEV void softmax_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

template <typename T> constexpr uint32_t idesc(int M) {
  return (std::is_same<T, __nv_bfloat16>::value ? tc::idesc_bf16(M, N) : tc::idesc_bf16(M, N) & ~((1u << 7) | (1u << 10)));
}

// the unit that follows; true at the end of the share's part of the current one
S0_DEV bool step(Cur& c, const KvAttnArgs& a) {
  if (++c.t < c.n) return false;
  c.t = 0;
  cur_next_unit(c, a, KT);
  return true;
}

// sums (maxima) over a warp's lanes of v[0..31]: lane i ends with that of v[i]
template <bool MAX> S0_DEV float transpose_reduce(float* v, int lane) {
#pragma unroll
  for (int w = 16; w > 0; w >>= 1) {
    const bool up = lane & w;
#pragma unroll
    for (int i = 0; i < w; ++i) {
      const float mine = up ? v[i + w] : v[i], got = __shfl_xor_sync(0xffffffffu, up ? v[i] : v[i + w], w);
      v[i] = MAX ? fmaxf(mine, got) : mine + got;
    }
  }
  return v[0];
}

template <typename T, int HD>
__global__ void __launch_bounds__(NT, 1) kv_attn_t5_k(KvAttnArgs a, int ctas) {
  using RG = Ring<HD>;
  using SM = Smem<HD>;
  constexpr int SLOTS = RG::SLOTS;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024 - (tc::smem_u32(smem_raw) & 1023)) & 1023);
  unsigned char *sQ = smem + SM::Q, *sP = smem + SM::P;
  float* s_m = reinterpret_cast<float*>(smem + SM::F);             // [N] references
  float* s_al = s_m + N;                                          // [N] factors, later 1 / sum
  float* s_l = s_al + N;                                          // [4][N] partial sums or maxima of the warps
  uint32_t* s_vis = reinterpret_cast<uint32_t*>(s_l + 4 * N);      // [2][2][KT] rows that see a key, 32 bits each
  Bars& bars = *reinterpret_cast<Bars*>(s_vis + 4 * KT);
  volatile int* abort = &bars.abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int R = a.T * a.group;
  join_may_start();

  if (warp == ST / 32) tc::tmem_alloc(&bars.tslot, TM_COLS);
  if (tid == 0) {
    for (int i = 0; i < SLOTS; ++i) {
      tc::mbar_init(&bars.full[i], LT);
      tc::mbar_init(&bars.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&bars.sfull[i], 1);
      tc::mbar_init(&bars.sempty[i], ST);
      tc::mbar_init(&bars.qempty[i], 1);
    }
    tc::mbar_init(&bars.pfull, ST);
    tc::mbar_init(&bars.pdone, 1);
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&bars.mfull[i], 32);
      tc::mbar_init(&bars.mempty[i], ST);
    }
    tc::mbar_init(&bars.drain, 1);
    bars.abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  Cur cur;
  const int share = (int)cta_share(cur, a, KT, reinterpret_cast<int*>(smem), ctas);   // scratch: the ring
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = bars.tslot;

  if (warp == NT / 32 - 1) {
    // ---- the new tokens of the units that this CTA ends ---------------------------------------------
    Cur c = cur;
    int tails = 0;
    bool ok = true;
    for (int i = 0; i < share && ok;) {
      const int h = c.u / a.nrb, rb = c.u - h * a.nrb, r0 = rb * N, ncache = (c.len + KT - 1) / KT;
      const int t1 = min(c.n, c.t + (share - i)), from = max(c.t, ncache) - ncache;
      const T *kn = (const T*)a.kn + c.b * a.kn_b + h * a.kn_h, *vn = (const T*)a.vn + c.b * a.vn_b + h * a.vn_h;
      T* kc = (T*)a.kc + c.b * a.kc_b + h * a.kc_h + c.len * a.kc_s;
      T* vc = (T*)a.vc + c.b * a.vc_b + h * a.vc_h + c.len * a.vc_s;
      // rows [j0, j0 + n) of the new ones, behind the cached ones as far as they fit; true: one is not finite
      auto copy = [&](const T* src, long ss, T* dst, long ds, int j0, int n, bool put) {
        constexpr int C = HD / 8, RP = 32 / C, U = 16;             // chunks of a row, rows of a pass, passes in flight
        const int ch = lane % C, fit = put ? a.S - c.len - j0 : 0;
        bool bad = false;
        src += (j0 + lane / C) * ss + ch * 8;
        dst += (j0 + lane / C) * ds + ch * 8;
        if (ch * 8 < a.hd)
#pragma unroll 1
          for (int j = lane / C; j < n; j += U * RP) {
            uint4 x[U];
#pragma unroll
            for (int k = 0; k < U; ++k)
              if (j + k * RP < n) x[k] = *reinterpret_cast<const uint4*>(src + k * RP * ss);
#pragma unroll
            for (int k = 0; k < U; ++k)
              if (j + k * RP < n) {
                bad |= any_inf<T>(x[k]);
                if (j + k * RP < fit) *reinterpret_cast<uint4*>(dst + k * RP * ds) = x[k];
              }
            src += U * RP * ss;
            dst += U * RP * ds;
          }
        __syncwarp();
        return __any_sync(0xffffffffu, bad);
      };
      for (int tt = from; tt < t1 - ncache; ++tt, ++tails) {
        const int j0 = tt * KT, n = min(KT, a.T - j0), buf = tails & 1;
        ok = __all_sync(0xffffffffu, wait(&bars.mempty[buf], ((tails >> 1) & 1) ^ 1, abort, a.wait_ns));   // the warp leaves as one
        if (!ok) break;
#pragma unroll 1
        for (int w = 0; w < 2 * KT / 32; ++w) {                    // 32 keys x 32 rows
          const int k0 = j0 + (w & (KT / 32 - 1)) * 32, key = k0 + lane, q0 = r0 + w / (KT / 32) * 32;
          if (k0 >= a.T) continue;                                 // no such keys: nobody looks
          const uint32_t v = q0 < R ? sees<32>(a, c.b, key, R, [=](int x) { return q0 + x; }) : 0u;
          s_vis[(buf * 2 * KT) + w * 32 + lane] = v;
        }
        const bool bad = copy(vn, a.vn_t, vc, a.vc_s, j0, n, rb == 0);
        if (lane == 0) bars.bad[buf] = bad;
        tc::mbar_arrive(&bars.mfull[buf]);
        if (rb == 0) {
          copy(kn, a.kn_t, kc, a.kc_s, j0, n, true);
          if (a.positions)
            for (int j = j0 + lane; j < min(j0 + n, a.S - c.len); j += 32)
              a.positions[c.b * a.pos_b + h * a.pos_h + c.len + j] = a.seen[c.b] + j;
        }
      }
      i += t1 - c.t;
      c.t = 0;
      cur_next_unit(c, a, KT);
    }
  } else if (warp > ST / 32) {
    // ---- loading --------------------------------------------------------------------------------
    constexpr int C = HD / 8, RS = LT / C;                         // 16-byte chunks of a row, rows of a pass (4 or 8)
    const int lt = tid - ST - 32, ch = lt % C, r0 = lt / C;
    const bool in = ch * 8 < a.hd;
    // where a chunk of pass x goes: two swizzles take turns where a pass is four rows
    const uint32_t off0 = (ch >> 3) * PANEL + r0 * 128 + (((ch & 7) ^ (r0 & 7)) << 4);
    const uint32_t off1 = (ch >> 3) * PANEL + r0 * 128 + (((ch & 7) ^ ((r0 + RS) & 7)) << 4);
    Cur c = cur;
    int n = 0, unit = 0;
    bool ok = true, fresh = true;
    for (int i = 0; i < share && ok; ++i) {
      const int h = c.u / a.nrb, rb = c.u - h * a.nrb, ncache = (c.len + KT - 1) / KT;
      const bool tail = c.t >= ncache;
      const int k0 = (tail ? c.t - ncache : c.t) * KT, rows = (tail ? a.T : c.len) - k0;
      if (fresh) {                                                 // a unit's queries come with its first keys
        ok = wait(&bars.qempty[unit & 1], ((unit >> 1) & 1) ^ 1, abort, a.wait_ns);
        if (!ok) break;
        for (int r = r0; r < N; r += RS) {
          const int row = rb * N + r, tok = div_group(a, row);
          const bool is = in && row < R;
          const T* p = (const T*)a.q + c.b * a.q_b + tok * a.q_t + (long)(h * a.group + row - tok * a.group) * a.q_h + ch * 8;
          cp_async16(sQ + (unit & 1) * SM::QB + (ch >> 3) * (N * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4), is ? p : a.q, is ? 16 : 0);
        }
      }
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        ok = wait(&bars.empty[n % SLOTS], ((n / SLOTS) & 1) ^ 1, abort, a.wait_ns);
        if (!ok) break;
        const long rs = v ? (tail ? a.vn_t : a.vc_s) : (tail ? a.kn_t : a.kc_s);
        const T* src = v ? (tail ? (const T*)a.vn + c.b * a.vn_b + h * a.vn_h : (const T*)a.vc + c.b * a.vc_b + h * a.vc_h)
                         : (tail ? (const T*)a.kn + c.b * a.kn_b + h * a.kn_h : (const T*)a.kc + c.b * a.kc_b + h * a.kc_h);
        src += (long)(k0 + r0) * rs + ch * 8;
        unsigned char* dst = smem + (n % SLOTS) * RG::SLOT;
        int more = in ? rows - r0 : 0;                             // a short loop: unrolled, it is bound by its own fetching
#pragma unroll 4
        for (int x = 0; x < KT / RS; ++x) {
          cp_async16(dst + (x & 1 ? off1 : off0), more > 0 ? src : (const T*)a.q, more > 0 ? 16 : 0);
          dst += RS * 128;
          src += RS * rs;
          more -= RS;
        }
        tc::cp_async_mbar_arrive(&bars.full[n % SLOTS]);           // once these copies have landed
        ++n;
      }
      fresh = step(c, a);
      unit += fresh;
    }
    cp_async_wait_all();
  } else if (warp == ST / 32) {
    // ---- the products ---------------------------------------------------------------------------
    if (lane == 0 && share > 0) {
      constexpr uint32_t id_s = idesc<T>(128), id_o = idesc<T>(HD) | tc::IDESC_A_MN | tc::IDESC_B_MN;
      Cur c = cur;
      bool ok = true, first = true, prev_first = true;
      int unit = 0;
      for (int i = 0; i <= share && ok; ++i) {
        if (i < share) {                                           // S^T of tile i
          const int n = 2 * i;
          ok = wait(&bars.full[n % SLOTS], (n / SLOTS) & 1, abort, a.wait_ns) && wait(&bars.sempty[i & 1], ((i >> 1) & 1) ^ 1, abort, a.wait_ns);
          if (!ok) break;
          tc::fence_proxy_async();                                 // the loaders' copies, for the products
          tc::fence_after_sync();
          const unsigned char *k = smem + (n % SLOTS) * RG::SLOT, *q = sQ + (unit & 1) * SM::QB;
#pragma unroll
          for (int x = 0; x < HD / 16; ++x)
            tc::mma_bf16(tmem + (i & 1) * N, tc::desc_sw128(k + (x >> 2) * PANEL, x & 3), tc::desc_sw128(q + (x >> 2) * (N * 128), x & 3), id_s, x > 0);
          tc::commit(&bars.empty[n % SLOTS]);
          tc::commit(&bars.sfull[i & 1]);
        }
        if (i > 0) {                                               // O^T of tile i - 1
          const int n = 2 * (i - 1) + 1;
          ok = wait(&bars.pfull, (i - 1) & 1, abort, a.wait_ns) && wait(&bars.full[n % SLOTS], (n / SLOTS) & 1, abort, a.wait_ns);
          if (!ok) break;
          tc::fence_proxy_async();
          tc::fence_after_sync();
          const unsigned char* v = smem + (n % SLOTS) * RG::SLOT;
#pragma unroll
          for (int x = 0; x < KT / 16; ++x)
            tc::mma_bf16(tmem + TM_O, tc::desc_mn_sw128(v + x * 2048, PANEL), tc::desc_mn_sw128(sP + x * 2048, PANEL), id_o, x > 0 || !prev_first);
          tc::commit(&bars.empty[n % SLOTS]);
          tc::commit(&bars.pdone);
        }
        prev_first = first;
        if (i < share) {
          first = step(c, a);
          if (first) {
            tc::commit(&bars.qempty[unit & 1]);                    // all of the unit's S^T have been issued
            ++unit;
          }
        }
      }
      // nothing may be in flight when the tensor memory is given back
      tc::commit(&bars.drain);
      int none = 0;
      wait(&bars.drain, 0, &none, DRAIN_NS);
    }
    __syncwarp();
  } else {
    // ---- softmax: thread = key of the tile and half of the rows, then channel of the output ------------
    constexpr int W = N / 2;
    const int kt = tid & (KT - 1), half = tid / KT, quarter = warp & 3;
    const uint32_t quad = (uint32_t)(32 * quarter) << 16 | (uint32_t)(half * W);
    float *m_ = s_m + half * W, *al_ = s_al + half * W;
    bool dead = false, stop = false;                               // this thread's wait ran out; all threads leave
    int i = 0, tails = 0;                                          // tiles of the share so far, of new tokens
    while (i < share && !stop) {
      const int b = cur.b, h = cur.u / a.nrb, rb = cur.u - h * a.nrb, r0 = rb * N, q0 = r0 + half * W;
      const long bh = (long)b * a.nkv + h;
      const int t1 = min(cur.n, cur.t + (share - i)), ncache = (cur.len + KT - 1) / KT;
      bool bad = false;                                            // some new V is not finite
      float l[W];
#pragma unroll
      for (int c = 0; c < W; ++c) l[c] = 0.f;
      if (tid < N) s_m[tid] = UNSET;
      for (int tt = cur.t; tt < t1; ++tt, ++i) {
        const bool tail = tt >= ncache;
        const int k0 = (tail ? tt - ncache : tt) * KT, nk = min(KT, (tail ? a.T : cur.len) - k0), key = k0 + kt;
        dead |= !wait(&bars.sfull[i & 1], (i >> 1) & 1, abort, a.wait_ns);
        if (any_of(dead)) {
          stop = true;
          break;
        }
        tc::fence_after_sync();
        bool bad_tile = false;
        float s[W];
        tc::tmem_ld32(tmem + quad + (i & 1) * N, s);
        tc::fence_before_sync();
        tc::mbar_arrive(&bars.sempty[i & 1]);
        if (tail || nk < KT) {
          uint32_t vis = kt < nk ? ~0u : 0u;
          if (tail) {
            const int buf = tails & 1;
            dead |= !wait(&bars.mfull[buf], (tails >> 1) & 1, abort, a.wait_ns);
            vis &= s_vis[buf * 2 * KT + half * KT + kt];
            bad_tile = bars.bad[buf];
            tc::mbar_arrive(&bars.mempty[buf]);
            ++tails;
          }
#pragma unroll
          for (int c = 0; c < W; ++c)
            if (!(vis >> c & 1)) s[c] = -CUDART_INF_F;
        }
        if (a.scores && kt < nk) {
          float* p = a.scores + (bh * R + q0) * a.sp + (tail ? cur.len : 0) + key;
#pragma unroll
          for (int c = 0; c < W; ++c)
            if (q0 + c < R) p[c * a.sp] = s[c] * a.scale_log2;
        }
        // does a score pass its row's reference?
        float over = -CUDART_INF_F;
#pragma unroll
        for (int c = 0; c < W; c += 4) {
          const float4 m = *reinterpret_cast<const float4*>(m_ + c);
          over = fmaxf(over, fmaxf(fmaxf(s[c] - m.x, s[c + 1] - m.y), fmaxf(s[c + 2] - m.z, s[c + 3] - m.w)));
        }
        const bool move = any_of(over * a.scale_log2 > Ref<T>::lazy);
        if (i > 0) dead |= !wait(&bars.pdone, (i - 1) & 1, abort, a.wait_ns);  // P and O^T of the tile before are done with
        if (move) {
          float x[W];
#pragma unroll
          for (int c = 0; c < W; ++c) x[c] = s[c];
          s_l[quarter * N + half * W + lane] = transpose_reduce<true>(x, lane);
          softmax_sync();
          if (tid < N) {
            const float x = fmaxf(fmaxf(s_l[tid], s_l[N + tid]), fmaxf(s_l[2 * N + tid], s_l[3 * N + tid]));
            const float was = s_m[tid], now = fmaxf(was, x);
            s_al[tid] = ex2((was - now) * a.scale_log2);
            s_m[tid] = now;
          }
          softmax_sync();
#pragma unroll
          for (int c = 0; c < W; ++c) l[c] *= al_[c];
          if (tt > cur.t) {
            tc::fence_after_sync();
            float o[W];
            tc::tmem_ld32(tmem + quad + TM_O, o);
#pragma unroll
            for (int c = 0; c < W; ++c) o[c] *= al_[c];
            tc::tmem_st32(tmem + quad + TM_O, o);
            tc::tmem_wait_st();
            tc::fence_before_sync();
          }
        }
        // P^T: this key's probabilities, 32 of a row of 64
#pragma unroll
        for (int c = 0; c < W; c += 8) {
          const float4 m0 = *reinterpret_cast<const float4*>(m_ + c), m1 = *reinterpret_cast<const float4*>(m_ + c + 4);
          const float m[8] = {m0.x, m0.y, m0.z, m0.w, m1.x, m1.y, m1.z, m1.w};
          float p[8];
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            p[x] = ex2(fmaf(s[c + x] - m[x], a.scale_log2, Ref<T>::up));
            l[c + x] += p[x];
          }
          *reinterpret_cast<uint4*>(sP + kt * 128 + (((half * (W / 8) + (c >> 3)) ^ (kt & 7)) << 4)) =
              make_uint4(pack2<T>(p[0], p[1]), pack2<T>(p[2], p[3]), pack2<T>(p[4], p[5]), pack2<T>(p[6], p[7]));
        }
        bad |= bad_tile;
        if (bad_tile && half) {
          // what is not finite in V must not meet the zero probabilities of the rows that do not see it: it is
          // taken out of the tile here and added to the others' output at the end
          const int n = 2 * i + 1;
          dead |= !wait(&bars.full[n % SLOTS], (n / SLOTS) & 1, abort, a.wait_ns);
          unsigned short* v = reinterpret_cast<unsigned short*>(smem + (n % SLOTS) * RG::SLOT + kt * 128);
          for (int x = 0; x < HD; ++x) {
            unsigned short* e = v + (x >> 6) * (PANEL / 2) + (x & 63);
            if ((*e & Inf<T>::mask) == Inf<T>::mask) *e = 0;
          }
        }
        tc::fence_proxy_async();
        tc::fence_before_sync();
        tc::mbar_arrive(&bars.pfull);
      }
      if (stop) break;
      // ---- the unit's output ----------------------------------------------------------------------
      const bool first = cur.t == 0, all = first && t1 == cur.n;
      const long slot = 2L * blockIdx.x + (first ? 1 : 0);
      s_l[quarter * N + half * W + lane] = transpose_reduce<false>(l, lane);
      dead |= !wait(&bars.pdone, (i - 1) & 1, abort, a.wait_ns);
      if (any_of(dead)) break;
      if (tid < N) {
        const float x = (s_l[tid] + s_l[N + tid]) + (s_l[2 * N + tid] + s_l[3 * N + tid]);
        const float m = s_m[tid] == UNSET ? -CUDART_INF_F : s_m[tid] * a.scale_log2;
        s_al[tid] = !all ? Ref<T>::down : x == 0.f ? 0.f : 1.f / x;
        if (r0 + tid < R) {
          if (!all) *reinterpret_cast<float2*>(a.part_ml + (slot * a.rows + tid) * 2) = make_float2(m, x * Ref<T>::down);
          else if (a.norm) reinterpret_cast<float2*>(a.norm)[bh * R + r0 + tid] = row_norm(m, x * Ref<T>::down);
        }
      }
      softmax_sync();
      tc::fence_after_sync();
      // 128 channels: lane = channel; 64: 16 channels in the first lanes of every quadrant
      const int d = HD == 128 ? kt : lane < 16 ? 16 * quarter + lane : HD;
      float o[W];
      tc::tmem_ld32(tmem + quad + TM_O, o);
      tc::fence_before_sync();
      if (bad && d < a.hd) {
        const T* vn = (const T*)a.vn + b * a.vn_b + h * a.vn_h + d;
        for (int j = 0; j < a.T; ++j) {
          const float x = Elem<T>::to(vn[j * a.vn_t]);
          const int tile = ncache + j / KT;
          if (isfinite(x) || tile < cur.t || tile >= t1) continue;
          const uint32_t v = sees<W>(a, b, j, R, [=](int c) { return q0 + c; });
#pragma unroll
          for (int c = 0; c < W; ++c)
            if (v >> c & 1) o[c] += x;
        }
      }
      if (all) {
        // through the P tile, which nothing reads now: whole rows leave in 16-byte pieces
        T* stage = reinterpret_cast<T*>(sP);
        if (d < HD) {
#pragma unroll
          for (int c = 0; c < W; ++c) stage[(half * W + c) * HD + d] = Elem<T>::of(o[c] * al_[c]);
        }
        softmax_sync();
        constexpr int C = HD / 8;
        for (int e = tid; e < N * C; e += ST) {
          const int row = r0 + e / C, x = e % C * 8, tok = div_group(a, row);
          if (row < R && x < a.hd)
            *reinterpret_cast<uint4*>((T*)a.o + (((long)b * a.T + tok) * a.nkv * a.group + h * a.group + row - tok * a.group) * a.hd + x) =
                *reinterpret_cast<const uint4*>(stage + e / C * HD + x);
        }
      } else if (d < a.hd) {
        float* p = a.part_o + (slot * a.rows + half * W) * a.hd + d;
#pragma unroll
        for (int c = 0; c < W; ++c) {
          if (q0 + c < R) *p = o[c] * Ref<T>::down;
          p += a.hd;
        }
      }
      softmax_sync();                                              // s_m, s_al, s_l and the P tile have been read
      cur.t = 0;
      cur_next_unit(cur, a, KT);
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  if (warp == ST / 32) tc::tmem_dealloc(tmem, TM_COLS);
  if (bars.abort) {                                                // all threads read the same: nobody writes it any more
    // No output of this CTA can be told from memory that was never written: all of its rows become NaN, whole units
    // here, pieces through their sums in the join.
    if (tid == 0) atomicExch(&gave_up, 1);
    const int tiles = (int)cta_share(cur, a, KT, reinterpret_cast<int*>(smem), ctas);
    for (int i = 0; i < tiles;) {
      const int h = cur.u / a.nrb, r0 = (cur.u - h * a.nrb) * N, nr = min(N, R - r0), t1 = min(cur.n, cur.t + (tiles - i));
      if (cur.t == 0 && t1 == cur.n) {
        for (int e = tid; e < nr * a.hd; e += NT) {
          const int row = r0 + e / a.hd, tok = div_group(a, row);
          ((T*)a.o)[(((long)cur.b * a.T + tok) * a.nkv * a.group + h * a.group + row - tok * a.group) * a.hd + e % a.hd] = Elem<T>::of(CUDART_NAN_F);
        }
        if (a.norm)
          for (int r = tid; r < nr; r += NT) reinterpret_cast<float2*>(a.norm)[((long)cur.b * a.nkv + h) * R + r0 + r] = make_float2(0.f, CUDART_NAN_F);
      } else {
        for (int r = tid; r < nr; r += NT)
          *reinterpret_cast<float2*>(a.part_ml + ((2L * blockIdx.x + (cur.t == 0 ? 1 : 0)) * a.rows + r) * 2) = make_float2(0.f, CUDART_NAN_F);
      }
      i += t1 - cur.t;
      cur.t = 0;
      cur_next_unit(cur, a, KT);
    }
  }
}

template <typename T, int HD>
int run(const KvAttnArgs& a, cudaStream_t st) {
  const size_t sm = Smem<HD>::BYTES;
  const cudaError_t e = cudaFuncSetAttribute(kv_attn_t5_k<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sm);
  if (e != cudaSuccess) return (int)e;
  kv_attn_t5_k<T, HD><<<a.whole ? a.B * a.nkv * a.nrb : a.ctas, NT, sm, st>>>(a, a.ctas);
  return launched();
}

}  // namespace t5
}  // namespace kv
}  // namespace s0

int kv_status_word(int** word) { return (int)cudaGetSymbolAddress((void**)word, s0::kv::t5::gave_up); }

// takes what kv_attn_tc_takes accepts
void kv_attn_t5_plan(KvAttnArgs& a, int sms) {
  using namespace s0::kv::t5;
  a.tc = 2;
  a.rows = N;
  a.nrb = (a.T * a.group + N - 1) / N;
  a.tile = KT;
  a.ctas = sms;
  a.min_per = 1;
  a.whole = 0;
  a.extra = 8;
  a.least = 20;
}

int kv_attn_t5_launch(const KvAttnArgs& a, int dtype, cudaStream_t st) {
  using namespace s0::kv::t5;
  if (dtype == 1) return a.hd > 64 ? run<__half, 128>(a, st) : run<__half, 64>(a, st);
  return a.hd > 64 ? run<__nv_bfloat16, 128>(a, st) : run<__nv_bfloat16, 64>(a, st);
}
