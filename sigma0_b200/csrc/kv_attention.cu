// Attention of a few new tokens over a key / value cache: the fp32 kernel for any element
// type, head size up to 512 and alignment, and the kernel that joins the pieces of a split (kv_attention_tc.cu has the
// tensor-core kernel for aligned 16-bit caches).
//
// Row r = (new token t, query head g of the key head's group) attends to the len cached keys and
// to the new tokens that its mask row sees:
//   s_rj = scale q_r . k_j,   o_r = sum_j p_rj v_j,   p_rj = exp(s_rj - max_j) / sum_j exp(...)
// in one pass over the keys with a running maximum and sum.  The new tokens' keys and values are
// read from their own tensors and stored behind the cached ones on the way.  A row that sees
// nothing gives zeros.  With weights, sum_r p_rj is added to the slot of key j: the scores (base 2,
// scaled) are kept in a scratch tensor, since p needs the row's final maximum and sum.
#include <algorithm>

#include "kv_attention.cuh"

namespace s0 {
namespace kv {

// warps of a block: wide heads leave one block on an SM
template <int HDP> constexpr int simt_warps() { return HDP == 512 ? 8 : 4; }

S0_DEV void prefetch(const void* p) { asm volatile("prefetch.global.L1 [%0];" ::"l"(p)); }
// two fp32 products and sums in one instruction
S0_DEV unsigned long long fma2(unsigned long long x, unsigned long long y, unsigned long long z) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
  return r;
}

// Keys of a slab: one per lane (64 channels), or per 2, 4 or 8 lanes that share its channels.  Its rows lie
// lane_parts * 4 words apart modulo 32 banks, so that the 8 lanes of a 16-byte access hit different banks.
template <int HDP> constexpr int lane_parts() { return HDP / 64; }
template <int HDP> constexpr int slab_keys() { return 32 / lane_parts<HDP>(); }
template <int HDP> constexpr int slab_ld() { return HDP + 4 * lane_parts<HDP>(); }
template <int HDP> constexpr int most_rows() { return HDP == 64 ? 32 : HDP == 128 ? 16 : 8; }
template <int HDP, int RB> constexpr size_t simt_bytes() {
  return 4 * ((size_t)simt_warps<HDP>() * 2 * slab_keys<HDP>() * slab_ld<HDP>()   // K and V slabs
              + RB * HDP                                          // queries
              + simt_warps<HDP>() * RB * (slab_keys<HDP>() + 4)                   // probabilities
              + 2 * RB * (HDP + 2));                               // two warps' results
}

// HDP: the head size padded to 64, 128, 256 or 512; RB: rows of a block; a.vec: 16-byte rows of floats.
//
// Every warp streams slabs of keys of its own (kv_attention_tc.cu does the same).  Scores: a lane holds
// its key's channels in registers and reads the queries as broadcasts, 4 products per 16-byte load of
// shared memory and row.  Output: a lane owns HDP / 32 channels of all rows, reads V once and the
// probabilities as broadcasts.  K of the next slab is fetched while V is used and the other way round.
// What bounds it: HBM for few rows (one token, 8 contexts of up to 5,000, 16 x 128 floats: 86 us of a floor of 64), the
// issue of fp32 products from some 16 rows on (22 rows over 8 contexts of up to 2,200, 16 x 64: 90 us of 15; 41% of the
// issue slots at the two warps per scheduler that 250 registers leave).
template <typename T, int HDP, int RB>
__global__ void __launch_bounds__(32 * simt_warps<HDP>(), HDP == 512 ? 1 : 2) kv_attn_any_k(KvAttnArgs a, int ctas) {
  constexpr int SW = simt_warps<HDP>();
  constexpr int DL = lane_parts<HDP>(), NK = slab_keys<HDP>(), LD = slab_ld<HDP>(), PL = NK + 4;
  constexpr int COLS = HDP / 32, RG = RB < 4 ? RB : 4;             // channels of a lane; rows at a time in the scores
  constexpr int KH = HDP / DL / 4;                                 // 16-byte groups of channels of a lane
  constexpr int JS = COLS > 8 ? 2 : 4;                             // keys at a time in the output
  extern __shared__ __align__(16) float s_f[];
  join_may_start();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, kl = lane / DL, dl = lane % DL;
  const int R = a.T * a.group;
  float* sK = s_f + warp * 2 * NK * LD;
  float* sV = sK + NK * LD;
  float* sQ = s_f + SW * 2 * NK * LD;                              // [RB][HDP], scaled
  float* sP = sQ + RB * HDP + warp * RB * PL;                      // [RB][PL]
  float* sJ = sQ + RB * HDP + SW * RB * PL;                        // [2][RB][HDP]
  float* sM = sJ + 2 * RB * HDP;                                   // [2][RB][2]
  Cur cur;
  const long share = cta_share(cur, a, NK, reinterpret_cast<int*>(s_f), ctas);
  __syncthreads();
  if (share <= 0) return;
  for (int i = tid; i < SW * 2 * NK * LD; i += 32 * SW) s_f[i] = 0.f;   // channels past hd stay 0
  __syncthreads();

  Cur ahead = cur;
  int left = (int)((share - warp + SW - 1) / SW);
  if (left > 0) cur_skip(ahead, a, NK, warp);
  // rows of K (then V) of the next slab; a row that does not exist becomes 0
  auto fetch = [&](float* dst, bool value) {
    if (left > 0) {
      const int ncache = (ahead.len + NK - 1) / NK, h = ahead.u / a.nrb;
      const bool tail = ahead.t >= ncache;
      const int k0 = (tail ? ahead.t - ncache : ahead.t) * NK, rows = (tail ? a.T : ahead.len) - k0;
      const long rs = value ? (tail ? a.vn_t : a.vc_s) : (tail ? a.kn_t : a.kc_s);
      const T* src = (value ? (tail ? (const T*)a.vn + ahead.b * a.vn_b + h * a.vn_h : (const T*)a.vc + ahead.b * a.vc_b + h * a.vc_h)
                            : (tail ? (const T*)a.kn + ahead.b * a.kn_b + h * a.kn_h : (const T*)a.kc + ahead.b * a.kc_b + h * a.kc_h)) +
                     (long)k0 * rs;
      if constexpr (sizeof(T) == 4) {
        if (a.vec) {
          constexpr int C = HDP / 4, L = C < 32 ? C : 32;          // groups of a row, lanes on a row
#pragma unroll
          for (int r = lane / L; r < NK; r += 32 / L)
#pragma unroll
            for (int c = lane % L; c < C; c += L)
              if (c * 4 < a.hd) cp_async16(dst + r * LD + c * 4, r < rows ? src + r * rs + c * 4 : src, r < rows ? 16 : 0);
        } else {
          for (int r = 0; r < NK; ++r)
            for (int d = lane; d < a.hd; d += 32) cp_async4(dst + r * LD + d, r < rows ? src + r * rs + d : src, r < rows ? 4 : 0);
        }
      } else {
        // element loads (odd alignments): 32 in flight per lane, or the slab waits for one trip after another
        constexpr int CPL = HDP / 32, RU = 32 / CPL < NK ? 32 / CPL : NK;
#pragma unroll 1
        for (int r = 0; r < NK; r += RU) {
          T x[RU][CPL];
#pragma unroll
          for (int y = 0; y < RU; ++y)
#pragma unroll
            for (int k = 0; k < CPL; ++k)
              x[y][k] = r + y < rows && lane + 32 * k < a.hd ? src[(r + y) * rs + lane + 32 * k] : Elem<T>::of(0.f);
#pragma unroll
          for (int y = 0; y < RU; ++y)
#pragma unroll
            for (int k = 0; k < CPL; ++k)
              if (lane + 32 * k < a.hd) dst[(r + y) * LD + lane + 32 * k] = Elem<T>::to(x[y][k]);
        }
      }
      if (value && --left > 0) {
        cur_skip(ahead, a, NK, SW);
        if constexpr (sizeof(T) == 2) {
          // element loads are waited for: the lines of the slab after this one (32 of K, 32 of V) are on their way before
          constexpr int LR = HDP / 64;                             // lines of a row
          const int r = ahead.t * NK + lane / LR, at = lane % LR * 64, hh = ahead.u / a.nrb;
          if (r < ahead.len && at < a.hd) {
            prefetch((const T*)a.kc + ahead.b * a.kc_b + hh * a.kc_h + (long)r * a.kc_s + at);
            prefetch((const T*)a.vc + ahead.b * a.vc_b + hh * a.vc_h + (long)r * a.vc_s + at);
          }
        }
      }
    }
    cp_async_commit();
  };
  fetch(sK, false);
  fetch(sV, true);

  long done = 0, mine = warp;
  while (done < share) {
    const int b = cur.b, h = cur.u / a.nrb, rb = cur.u - h * a.nrb, r0 = rb * RB, nr = min(RB, R - r0);
    const long bh = (long)b * a.nkv + h;
    const int t1 = (int)min((long)cur.n, cur.t + (share - done));
    const int ncache = (cur.len + NK - 1) / NK;
    const long end = done + (t1 - cur.t);
    __syncthreads();                                               // the last unit's queries have been read
    constexpr int QN = RB * HDP / (32 * SW) > 0 ? RB * HDP / (32 * SW) : 1, QB = QN < 8 ? QN : 8;   // loads in flight
    for (int i0 = tid; i0 < RB * HDP; i0 += 32 * SW * QB) {
      float x[QB];
#pragma unroll
      for (int k = 0; k < QB; ++k) {
        const int i = i0 + 32 * SW * k, r = i / HDP, d = i % HDP, tok = div_group(a, r0 + r);
        x[k] = r < nr && d < a.hd ? Elem<T>::to(((const T*)a.q)[b * a.q_b + tok * a.q_t + (long)(h * a.group + r0 + r - tok * a.group) * a.q_h + d]) : 0.f;
      }
#pragma unroll
      for (int k = 0; k < QB; ++k)
        if (i0 + 32 * SW * k < RB * HDP) sQ[i0 + 32 * SW * k] = x[k] * a.scale_log2;
    }
    if (t1 == cur.n && rb == 0) {                                  // the new rows go behind the cached ones
      constexpr int U = 8;                                         // rows in flight per warp
      const T* kn = (const T*)a.kn + b * a.kn_b + h * a.kn_h;
      const T* vn = (const T*)a.vn + b * a.vn_b + h * a.vn_h;
      T* kc = (T*)a.kc + b * a.kc_b + h * a.kc_h + cur.len * a.kc_s;
      T* vc = (T*)a.vc + b * a.vc_b + h * a.vc_h + cur.len * a.vc_s;
      const int fit = min(a.T, a.S - cur.len);
      for (int d = lane; d < a.hd; d += 32)
        for (int r = warp; r < fit; r += U * SW) {
          T x[U], y[U];
#pragma unroll
          for (int i = 0; i < U; ++i)
            if (r + i * SW < fit) {
              x[i] = kn[(r + i * SW) * a.kn_t + d];
              y[i] = vn[(r + i * SW) * a.vn_t + d];
            }
#pragma unroll
          for (int i = 0; i < U; ++i)
            if (r + i * SW < fit) {
              kc[(r + i * SW) * a.kc_s + d] = x[i];
              vc[(r + i * SW) * a.vc_s + d] = y[i];
            }
        }
      if (a.positions)
        for (int r = tid; r < fit; r += 32 * SW) a.positions[b * a.pos_b + h * a.pos_h + cur.len + r] = a.seen[b] + r;
    }
    __syncthreads();
    float o[RB][COLS];
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
      for (int c = 0; c < COLS; ++c) o[r][c] = 0.f;
    float m = -CUDART_INF_F, l = 0.f;                              // of row `lane`

    for (; mine < end; mine += SW) {
      const int tt = cur.t + (int)(mine - done);
      const bool tail = tt >= ncache;
      const int k0 = (tail ? tt - ncache : tt) * NK, nk = min(NK, (tail ? a.T : cur.len) - k0);
      cp_async_wait_group<1>();
      __syncwarp();
      // ---- scores, row group by row group --------------------------------------------------------
      float al = 1.f;                                              // rescaling of row `lane`
      bool moved = false;
#pragma unroll 1
      for (int rg = 0; rg < nr; rg += RG) {
        float s[RG];
        ulonglong2 k[KH];                                        // two pairs of channels
#pragma unroll
        for (int i = 0; i < KH; ++i) k[i] = *reinterpret_cast<const ulonglong2*>(sK + kl * LD + (dl + DL * i) * 4);
#pragma unroll
        for (int r = 0; r < RG; ++r) {
          unsigned long long x = 0, y = 0;
#pragma unroll
          for (int i = 0; i < KH; ++i) {
            const ulonglong2 q = *reinterpret_cast<const ulonglong2*>(sQ + (rg + r) * HDP + (dl + DL * i) * 4);
            x = fma2(q.x, k[i].x, x);
            y = fma2(q.y, k[i].y, y);
          }
          const float2 u = *reinterpret_cast<const float2*>(&x), v = *reinterpret_cast<const float2*>(&y);
          s[r] = (u.x + u.y) + (v.x + v.y);
        }
        bool far = false;
        uint32_t see = kl < nk ? ~0u : 0u;
        if (tail) see &= sees<RG>(a, b, k0 + kl, R, [=](int r) { return r0 + rg + r; });
#pragma unroll
        for (int r = 0; r < RG; ++r) {
          if (DL > 1) s[r] += __shfl_xor_sync(0xffffffffu, s[r], 1);
          if (DL > 2) s[r] += __shfl_xor_sync(0xffffffffu, s[r], 2);
          if (DL > 4) s[r] += __shfl_xor_sync(0xffffffffu, s[r], 4);
          if (!(see >> r & 1)) s[r] = -CUDART_INF_F;
          if (a.scores && dl == 0 && kl < nk && rg + r < nr)
            a.scores[(bh * R + r0 + rg + r) * a.sp + (tail ? cur.len : 0) + k0 + kl] = s[r];
          far |= s[r] > __shfl_sync(0xffffffffu, m, rg + r) + 8.f;
        }
        if (__any_sync(0xffffffffu, far)) {                        // the reference of a row moves (as on the tensor cores)
          moved = true;
#pragma unroll
          for (int r = 0; r < RG; ++r) {
            float x = fmaxf(s[r], __shfl_sync(0xffffffffu, m, rg + r));
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
            if (lane == rg + r && x != -CUDART_INF_F) {
              al = ex2(m - x);
              m = x;
            }
          }
        }
#pragma unroll
        for (int r = 0; r < RG; ++r) {
          const float x = __shfl_sync(0xffffffffu, m, rg + r);
          if (dl == 0) sP[(rg + r) * PL + kl] = ex2(s[r] - (x == -CUDART_INF_F ? 0.f : x));
        }
      }
      __syncwarp();
      fetch(sK, false);
      // ---- the row sums, row `lane` --------------------------------------------------------------
      if (lane < nr) {
        float x = 0.f, y = 0.f;
#pragma unroll
        for (int j = 0; j < NK; j += 4) {
          const float4 q = *reinterpret_cast<const float4*>(sP + lane * PL + j);
          x += q.x + q.y;
          y += q.z + q.w;
        }
        l = l * al + (x + y);
      }
      if (moved) {
#pragma unroll
        for (int r = 0; r < RB; ++r) {
          const float f = __shfl_sync(0xffffffffu, al, r);
#pragma unroll
          for (int c = 0; c < COLS; ++c) o[r][c] *= f;
        }
      }
      cp_async_wait_group<1>();
      __syncwarp();
      bool bad = false;
      if (tail) {
        // what is not finite must not meet the zero probabilities of rows that do not see it
        for (int i = lane * 4; i < NK * LD; i += 128) {
          const float4 x = *reinterpret_cast<const float4*>(sV + i);
          bad |= !(isfinite(x.x) && isfinite(x.y) && isfinite(x.z) && isfinite(x.w));
        }
        bad = __any_sync(0xffffffffu, bad);
        if (bad) {
          for (int i = lane; i < NK * LD; i += 32)
            if (!isfinite(sV[i])) sV[i] = 0.f;
          __syncwarp();
        }
      }
      // ---- output --------------------------------------------------------------------------------
#pragma unroll 1
      for (int j = 0; j < NK; j += JS) {
        float v[JS][COLS];
#pragma unroll
        for (int x = 0; x < JS; ++x) {
          if constexpr (COLS == 2) {
            *reinterpret_cast<float2*>(v[x]) = *reinterpret_cast<const float2*>(sV + (j + x) * LD + lane * 2);
          } else {
#pragma unroll
            for (int c = 0; c < COLS; c += 4)
              *reinterpret_cast<float4*>(v[x] + c) = *reinterpret_cast<const float4*>(sV + (j + x) * LD + lane * 4 + c * 32);
          }
        }
#pragma unroll
        for (int g = 0; g < RB; g += RG) {
          if (g >= nr) break;
#pragma unroll
          for (int r = g; r < g + RG; ++r) {
            float q[JS];
            if constexpr (JS == 4) *reinterpret_cast<float4*>(q) = *reinterpret_cast<const float4*>(sP + r * PL + j);
            else *reinterpret_cast<float2*>(q) = *reinterpret_cast<const float2*>(sP + r * PL + j);
#pragma unroll
            for (int x = 0; x < JS; ++x)
#pragma unroll
              for (int c = 0; c < COLS; ++c) o[r][c] = fmaf(q[x], v[x][c], o[r][c]);
          }
        }
      }
      if (bad) {
        const T* vn = (const T*)a.vn + b * a.vn_b + h * a.vn_h;
        for (int j = 0; j < nk; ++j) {
          const unsigned vis = __ballot_sync(0xffffffffu, lane < nr && sees<1>(a, b, k0 + j, R, [=](int) { return r0 + lane; }));
#pragma unroll
          for (int c = 0; c < COLS; ++c) {
            const int d = COLS == 2 ? lane * 2 + c : lane * 4 + (c & 3) + (c >> 2) * 128;
            const float x = d < a.hd ? Elem<T>::to(vn[(k0 + j) * a.vn_t + d]) : 0.f;
            if (isfinite(x)) continue;
#pragma unroll
            for (int r = 0; r < RB; ++r)
              if (vis >> r & 1) o[r][c] += x;
          }
        }
      }
      __syncwarp();
      fetch(sV, true);
    }

    // ---- join the warps: the last two hand over to the two before, and so on; then 1 to 0 ----------
    auto give = [&](int slot) {
#pragma unroll
      for (int r = 0; r < RB; ++r)
#pragma unroll
        for (int c = 0; c < COLS; ++c) sJ[((slot * RB + r) * COLS + c) * 32 + lane] = o[r][c];
      if (lane < RB) {
        sM[(slot * RB + lane) * 2] = m;
        sM[(slot * RB + lane) * 2 + 1] = l;
      }
    };
    auto take = [&](int slot) {
      float e0 = 1.f, e1 = 0.f;
      if (lane < RB) {
        const float m2 = sM[(slot * RB + lane) * 2], x = fmaxf(m, m2);
        if (x != -CUDART_INF_F) {
          e0 = ex2(m - x);
          e1 = ex2(m2 - x);
        }
        m = x;
        l = l * e0 + sM[(slot * RB + lane) * 2 + 1] * e1;
      }
#pragma unroll
      for (int r = 0; r < RB; ++r) {
        const float f0 = __shfl_sync(0xffffffffu, e0, r), f1 = __shfl_sync(0xffffffffu, e1, r);
#pragma unroll
        for (int c = 0; c < COLS; ++c) o[r][c] = o[r][c] * f0 + sJ[((slot * RB + r) * COLS + c) * 32 + lane] * f1;
      }
    };
#pragma unroll 1
    for (int top = SW - 2; top >= 2; top -= 2) {
      if (warp / 2 * 2 == top) give(warp & 1);
      __syncthreads();
      if (warp / 2 * 2 == top - 2) take(warp & 1);
      __syncwarp();
      if (top > 2) __syncthreads();
    }
    if (warp == 1) give(1);                                        // only this warp has read slot 1
    __syncthreads();
    if (warp == 0) {
      take(1);
      const bool first = cur.t == 0, all = first && t1 == cur.n;
      const long slot = 2L * blockIdx.x + (first ? 1 : 0);
      const float inv = l == 0.f ? 0.f : 1.f / l;
      if (lane < nr) {
        if (all && a.norm) reinterpret_cast<float2*>(a.norm)[bh * R + r0 + lane] = row_norm(m, l);
        if (!all) *reinterpret_cast<float2*>(a.part_ml + (slot * a.rows + lane) * 2) = make_float2(m, l);
      }
#pragma unroll
      for (int r = 0; r < RB; ++r) {
        const float f = __shfl_sync(0xffffffffu, inv, r);
        if (r >= nr) continue;
        const int tok = div_group(a, r0 + r);
        T* po = (T*)a.o + (((long)b * a.T + tok) * a.nkv * a.group + h * a.group + r0 + r - tok * a.group) * a.hd;
        float* pp = a.part_o + (slot * a.rows + r) * a.hd;
#pragma unroll
        for (int c = 0; c < COLS; ++c) {
          const int d = COLS == 2 ? lane * 2 + c : lane * 4 + (c & 3) + (c >> 2) * 128;
          if (d >= a.hd) continue;
          if (all) po[d] = Elem<T>::of(o[r][c] * f);
          else pp[d] = o[r][c];
        }
      }
    }
    done = end;
    cur.t = 0;
    cur_next_unit(cur, a, NK);
  }
}

// Joins the pieces of the units that several CTAs share, and adds up the weights (64 books of up to
// 11,000 slots, one row: 28 MB of scores and 56 MB of weights in 25-30 us, most of it latency).  Blocks
// [0, row_blocks): rows of the output; the others: JT PER slots of one (sequence, key head) each.
constexpr int JT = 256;
// slots of a thread and rows at a time: one row wants many slots in flight, many rows share fewer
constexpr int slots_of(int rows) { return rows < 4 ? 8 : 4; }

struct Pieces {
  long c0, c1;  // first and last CTA of the unit
};
// piece of CTA c: see kv_attention.cuh
S0_DEV long piece(const KvAttnArgs& a, const Pieces& p, long c, int r) { return (2 * c + (c == p.c0 ? 1 : 0)) * a.rows + r; }
// one warp: maximum and sum of a row over its pieces
S0_DEV void row_sum(const KvAttnArgs& a, const Pieces& p, int r, float& M, float& L) {
  const int lane = threadIdx.x & 31;
  M = -CUDART_INF_F;
  L = 0.f;
  for (long c = p.c0 + lane; c <= p.c1; c += 32) M = fmaxf(M, a.part_ml[piece(a, p, c, r) * 2]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  const float base = M == -CUDART_INF_F ? 0.f : M;
  for (long c = p.c0 + lane; c <= p.c1; c += 32) {
    const long i = piece(a, p, c, r) * 2;
    L += a.part_ml[i + 1] * ex2(a.part_ml[i] - base);
  }
  L = warp_sum(L);
}

// WPR warps share the pieces of a row
template <typename T, int WPR, int PER>
__global__ void __launch_bounds__(JT) kv_join_k(KvAttnArgs a, int row_blocks) {
  constexpr int JW = JT * PER, UR = PER == 4 ? 4 : 1;
  constexpr int RPB = JT / 32 / WPR, COLS = 4;     // rows of a block, columns of a lane at a time
  __shared__ __align__(8) float s_x[JT * COLS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, R = a.T * a.group;
  const bool out = blockIdx.x < (unsigned)row_blocks;
  const int wb = blockIdx.x - row_blocks, nch = (a.S + a.T + JW - 1) / JW;
  const long total = (long)a.B * a.nkv * R, idx = (long)blockIdx.x * RPB + warp / WPR;
  const long bh = out ? min(idx, total - 1) / R : wb / nch;
  const int b = (int)(bh / a.nkv), h = (int)(bh - (long)b * a.nkv);
  join_wait();
  Plan plan{0, 1};
  int n = 1, surplus = 0;                           // costs of a row block, of them before its tiles
  long ub = 0;                                      // cost of the first tile of row block 0
  if (!a.whole) {
    plan = make_plan(a, a.prefix[a.B], a.ctas, a.min_per);
    const int p0 = a.prefix[b];
    n = a.prefix[b + 1] - p0;
    surplus = n - tiles_of(a, cached(a, b), a.tile);
    ub = (long)p0 * a.nkv * a.nrb + (long)h * a.nrb * n + surplus;
  }
  auto pieces = [&](int rb) {
    const long s = ub + (long)rb * n;
    return Pieces{s / plan.per, (s + n - surplus - 1) / plan.per};
  };
  if (out) {
    const int row = (int)(min(idx, total - 1) - bh * R), rb = row / a.rows, r = row - rb * a.rows;
    const Pieces p = pieces(rb);
    if ((WPR > 1 || idx < total) && p.c0 == p.c1) return;      // WPR > 1: one row in the block, all leave
    if (WPR == 1 && idx >= total) return;
    float M, L;
    row_sum(a, p, r, M, L);
    const float base = M == -CUDART_INF_F ? 0.f : M, inv = L == 0.f ? 0.f : 1.f / L;
    const int t = row / a.group, g = row - t * a.group;
    T* o = (T*)a.o + (((long)b * a.T + t) * a.nkv * a.group + h * a.group + g) * a.hd;
    for (int d0 = lane; d0 - lane < a.hd; d0 += 32 * COLS) {
      float x[COLS] = {};
#pragma unroll 4
      for (long c = p.c0 + warp % WPR; c <= p.c1; c += WPR) {
        const long i = piece(a, p, c, r);
        const float f = ex2(a.part_ml[i * 2] - base);
#pragma unroll
        for (int k = 0; k < COLS; ++k)
          if (d0 + 32 * k < a.hd) x[k] = fmaf(a.part_o[i * a.hd + d0 + 32 * k], f, x[k]);
      }
      if constexpr (WPR > 1) {
        __syncthreads();
#pragma unroll
        for (int k = 0; k < COLS; ++k) s_x[(warp * COLS + k) * 32 + lane] = x[k];
        __syncthreads();
        if (warp == 0) {
#pragma unroll
          for (int k = 0; k < COLS; ++k)
            for (int w = 1; w < WPR; ++w) x[k] += s_x[(w * COLS + k) * 32 + lane];
        }
      }
      if (WPR == 1 || warp == 0) {
#pragma unroll
        for (int k = 0; k < COLS; ++k)
          if (d0 + 32 * k < a.hd) o[d0 + 32 * k] = Elem<T>::of(x[k] * inv);
      }
    }
    return;
  }
  // weights: what does not depend on the row sums is loaded before they are known
  const int hi = min(a.S, cached(a, b) + a.T), j0 = (wb - (int)bh * nch) * JW;
  if (j0 >= hi) return;
  float* wt = a.weight + b * a.wt_b + h * a.wt_h + j0;
  const float* sc = a.scores + bh * R * a.sp + j0;
  float add[PER] = {}, was[PER], s[UR][PER];
  auto load = [&](int q0) {
#pragma unroll
    for (int q = 0; q < UR; ++q)
#pragma unroll
      for (int i = 0; i < PER; ++i)
        s[q][i] = q0 + q < R && j0 + i * JT + tid < hi ? sc[(q0 + q) * a.sp + i * JT + tid] : -CUDART_INF_F;
  };
#pragma unroll
  for (int i = 0; i < PER; ++i) was[i] = j0 + i * JT + tid < hi ? wt[i * JT + tid] : 0.f;
  load(0);
  for (int q0 = 0; q0 < R; q0 += JT) {
    __syncthreads();
    for (int q = warp; q < min(JT, R - q0); q += JT / 32) {
      const int row = q0 + q, rb = row / a.rows;
      const Pieces p = pieces(rb);
      float2 x;
      if (p.c0 == p.c1) {
        x = reinterpret_cast<const float2*>(a.norm)[bh * R + row];
      } else {
        float M, L;
        row_sum(a, p, row - rb * a.rows, M, L);
        x = row_norm(M, L);
      }
      if (lane == 0) *reinterpret_cast<float2*>(s_x + 2 * q) = x;
    }
    __syncthreads();
    for (int q = 0; q < min(JT, R - q0); q += UR) {
      float2 e[UR];
#pragma unroll
      for (int k = 0; k < UR; ++k) e[k] = q + k < JT && q0 + q + k < R ? *reinterpret_cast<const float2*>(s_x + 2 * (q + k)) : make_float2(0.f, 0.f);
      if (q0 + q > 0) load(q0 + q);
#pragma unroll
      for (int k = 0; k < UR; ++k)
#pragma unroll
        for (int i = 0; i < PER; ++i) add[i] = fmaf(ex2(s[k][i] - e[k].x), e[k].y, add[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (j0 + i * JT + tid < hi) wt[i * JT + tid] = was[i] + add[i];
}

template <typename T, int HDP, int RB>
int run_any(const KvAttnArgs& a, cudaStream_t st) {
  const size_t sm = std::max(simt_bytes<HDP, RB>(), (size_t)plan_ints(a.B) * 4);
  const cudaError_t e = cudaFuncSetAttribute(kv_attn_any_k<T, HDP, RB>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sm);
  if (e != cudaSuccess) return (int)e;
  kv_attn_any_k<T, HDP, RB><<<a.whole ? a.B * a.nkv * a.nrb : a.ctas, 32 * simt_warps<HDP>(), sm, st>>>(a, a.ctas);
  return launched();
}
template <typename T, int HDP>
int run_any_rows(const KvAttnArgs& a, cudaStream_t st) {
  if (a.rows == 1) return run_any<T, HDP, 1>(a, st);
  if constexpr (sizeof(T) == 4 && most_rows<HDP>() > 8) {
    if (a.rows > 8) return run_any<T, HDP, most_rows<HDP>()>(a, st);
  }
  return run_any<T, HDP, 8>(a, st);
}
template <typename T>
int launch(const KvAttnArgs& a, cudaStream_t st) {
  return a.hd <= 64 ? run_any_rows<T, 64>(a, st) : a.hd <= 128 ? run_any_rows<T, 128>(a, st)
         : a.hd <= 256 ? run_any_rows<T, 256>(a, st) : run_any_rows<T, 512>(a, st);
}

template <typename T, int PER>
int join_rows(const KvAttnArgs& a, cudaStream_t st) {
  // few rows leave room for a block each, whose warps take turns at the pieces
  const long rows = a.whole ? 0 : (long)a.B * a.nkv * a.T * a.group;
  const bool wide = rows > a.ctas;
  const long row_blocks = wide ? (rows + JT / 32 - 1) / (JT / 32) : rows;
  const long blocks = row_blocks + (a.weight ? (long)a.B * a.nkv * ((a.S + a.T + JT * PER - 1) / (JT * PER)) : 0);
  if (blocks == 0) return 0;                        // one CTA per unit and no weights: nothing is left to do
  return wide ? launch_after(kv_join_k<T, 1, PER>, (unsigned)blocks, JT, st, a, (int)row_blocks)
              : launch_after(kv_join_k<T, JT / 32, PER>, (unsigned)blocks, JT, st, a, (int)row_blocks);
}
template <typename T>
int join(const KvAttnArgs& a, cudaStream_t st) {
  return slots_of(a.T * a.group) == 8 ? join_rows<T, 8>(a, st) : join_rows<T, 4>(a, st);
}

}  // namespace kv
}  // namespace s0

long kv_launches() { return s0::kv::launches; }

void kv_attn_plan(KvAttnArgs& a, int dtype, int sms) {
  if (kv_attn_tc_takes(a, dtype)) return kv_attn_tc_plan(a, sms);
  a.tc = 0;
  using namespace s0::kv;
  const int R = a.T * a.group;
  const int most = dtype ? 8 : a.hd <= 64 ? most_rows<64>() : a.hd <= 128 ? most_rows<128>() : most_rows<256>();
  a.rows = R == 1 ? 1 : R <= 8 ? 8 : most;
  a.nrb = (R + a.rows - 1) / a.rows;
  a.tile = a.hd <= 64 ? slab_keys<64>() : a.hd <= 128 ? slab_keys<128>() : a.hd <= 256 ? slab_keys<256>() : slab_keys<512>();
  const int warps = a.hd > 256 ? simt_warps<512>() : simt_warps<64>();
  a.min_per = warps;
  a.whole = a.S + a.T <= 4 * a.tile * warps;
  a.extra = 8;
  a.least = 20;
  a.ctas = (a.hd > 256 ? 1 : 2) * sms;
  bool vec = dtype == 0 && a.hd % 4 == 0;
  for (long s : {a.kn_b, a.kn_t, a.kn_h, a.vn_b, a.vn_t, a.vn_h, a.kc_b, a.kc_h, a.kc_s, a.vc_b, a.vc_h, a.vc_s}) vec = vec && s % 4 == 0;
  for (const void* p : {a.kn, a.vn, (const void*)a.kc, (const void*)a.vc}) vec = vec && reinterpret_cast<uintptr_t>(p) % 16 == 0;
  a.vec = vec;
}

int kv_attn_launch(const KvAttnArgs& a, int dtype, cudaStream_t st) {
  if (a.B <= 0 || a.T <= 0) return 0;
  using namespace s0::kv;
  const int rc = a.tc ? kv_attn_tc_launch(a, dtype, st)
                 : dtype == 0 ? launch<float>(a, st) : dtype == 1 ? launch<__half>(a, st) : launch<__nv_bfloat16>(a, st);
  if (rc) return rc;
  return dtype == 0 ? join<float>(a, st) : dtype == 1 ? join<__half>(a, st) : join<__nv_bfloat16>(a, st);
}
