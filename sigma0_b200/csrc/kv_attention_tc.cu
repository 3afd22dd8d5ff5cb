// Attention of a few new tokens over a 16-bit key / value cache on the tensor cores (the operator is
// described in kv_attention.cu; heads up to 128 wide, 16-byte aligned rows).
//
// This kernel takes up to 16 rows (new tokens x query heads of a key head); more go to kv_attention_t5.cu.
// What bounds it: a step reads every cached key and value once and does 4 T group flops per element
// pair: HBM.  A CTA's tiles (see kv_attention.cuh) form one stream, whose loads run ahead by cp.async across the ends of
// units.
//
// The products are transposed: S^T = K Q^T and O^T = V^T P^T with mma.m16n8k16, so that the keys (then
// the channels) fill the 16 rows of the instruction and the queries its 8 columns.  One token of one
// head then wastes 7/8 of the products where the usual order wastes 15/16, a warp reads each K and V
// fragment once for all its 8 NT rows, and the accumulators are half as large.  P^T comes out as
// accumulators of the first product and goes into the second as its B operand; the two layouts are
// transposes of one another, which movmatrix turns.
// NT: column groups, 8 rows each.  Every warp takes slabs of its own, with a ring, a running maximum and a
// running sum of its own and no barrier among warps; they are joined at the end of a unit.
//
// Measured: one token of 64 books over up to 11,000 cached ones, 16 heads of 64: 290-300 us, 97% of the copy rate
// (with queries as the 16-row side: 430 us); one token over 66,000, 16 heads of 128: 84-87 us, the copy rate; without the
// join in both.
//
// The maximum that the exponentials refer to moves only when a score passes it by 2^8 (2^4 in fp16, whose range is
// short: see Ref in kv_attention.cuh): the probabilities may be that much larger, which changes no relative error, and
// the reduction over lanes and the rescaling of the output drop out of nearly every step.  p enters the second product as two numbers of the
// cache's type, its rounding and what that left (16 bits of a bf16 p, 22 of an fp16 one): HBM hides the second
// product (one token, 64 books: 322 us with and 319 us without it; 66,000 cached: 91.5 us both), and without it
// the error of one token is 1.4 times the output's own rounding.  The sum of the row is taken from the
// unrounded fp32 values.
#include <algorithm>

#include "kv_attention.cuh"

namespace s0 {
namespace kv {

template <typename T> S0_DEV void mma16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1);
template <> S0_DEV void mma16<__nv_bfloat16>(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) { mma_bf16(c, a, b0, b1); }
template <> S0_DEV void mma16<__half>(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// byte offset of 16-byte chunk c of row r in a tile of HD 16-bit channels: the chunks of eight
// consecutive rows fall into eight different groups of banks
template <int HD> S0_DEV int tile_at(int r, int c) { return r * HD * 2 + ((c ^ (r & 7)) << 4); }

S0_DEV uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// stores a slab of new rows behind the cached ones
template <typename T, int HD, int NK>
S0_DEV void put_slab(const char* st, const KvAttnArgs& a, int b, int h, int len, int k0, int nk, int i0, int step) {
  const int C = a.hd / 8;
  for (int i = i0; i < nk * C; i += step) {
    const int r = i / C, ch = i - r * C;
    const long at = len + k0 + r;
    if (at >= a.S) continue;
    *reinterpret_cast<uint4*>((T*)a.kc + b * a.kc_b + h * a.kc_h + at * a.kc_s + ch * 8) =
        *reinterpret_cast<const uint4*>(st + tile_at<HD>(r, ch));
    *reinterpret_cast<uint4*>((T*)a.vc + b * a.vc_b + h * a.vc_h + at * a.vc_s + ch * 8) =
        *reinterpret_cast<const uint4*>(st + NK * HD * 2 + tile_at<HD>(r, ch));
  }
  if (a.positions)
    for (int r = i0; r < nk; r += step)
      if (len + k0 + r < a.S) a.positions[b * a.pos_b + h * a.pos_h + len + k0 + r] = a.seen[b] + k0 + r;
}

constexpr int WARPS = 4, STAGES = 3, SLAB = 8192;   // warps, stages of a warp's ring, bytes of K and V in one

template <int HD> constexpr int slab_keys() { return SLAB / (HD * 4); }
// two warps' accumulators, maxima and sums in passing
template <int HD, int NT> constexpr int join_bytes() { return 2 * (HD / 16 * NT * 4 * 128 + NT * 8 * 2 * 4); }

template <typename T, int HD, int NT>
__global__ void __launch_bounds__(32 * WARPS, 2) kv_attn_tc_k(KvAttnArgs a, int ctas) {
  constexpr int NK = slab_keys<HD>();
  constexpr int KG = NK % 32 == 0 ? 2 : 1;                      // groups of 16 keys in flight at once
  constexpr int C = HD / 8, RS = 32 / C;                        // 16-byte chunks of a row, rows of a loading pass
  extern __shared__ __align__(128) char smem[];
  join_may_start();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int R = a.T * a.group;
  char* ring = smem + warp * STAGES * SLAB;
  float* sJ = reinterpret_cast<float*>(smem + WARPS * STAGES * SLAB);
  Cur cur;
  const long share = cta_share(cur, a, NK, reinterpret_cast<int*>(smem), ctas);
  __syncthreads();                                              // the plan's scratch becomes the rings
  if (share <= 0) return;

  // ---- loading: this warp's slabs of the share, ahead of their use -------------------------------
  Cur ahead = cur;
  int left = (int)((share - warp + WARPS - 1) / WARPS);
  const int ch = lane % C, lr = lane / C;                           // this thread's chunk and first row
  const bool in = ch * 8 < a.hd;
  const char *kp = nullptr, *vp = nullptr;                      // its first row's addresses in the slab
  long ks = 0, vs = 0;                                          // bytes from pass to pass
  int rows = 0;                                                 // rows of the source from the slab on
  bool fresh = false;                                           // the source is the new tokens
  auto aim = [&]() {
    const int ncache = (ahead.len + NK - 1) / NK, h = ahead.u / a.nrb;
    const bool tail = fresh = ahead.t >= ncache;
    const int k0 = (tail ? ahead.t - ncache : ahead.t) * NK;
    rows = (tail ? a.T : ahead.len) - k0;
    const long k1 = tail ? a.kn_t : a.kc_s, v1 = tail ? a.vn_t : a.vc_s;
    const T* k = tail ? (const T*)a.kn + ahead.b * a.kn_b + h * a.kn_h : (const T*)a.kc + ahead.b * a.kc_b + h * a.kc_h;
    const T* v = tail ? (const T*)a.vn + ahead.b * a.vn_b + h * a.vn_h : (const T*)a.vc + ahead.b * a.vc_b + h * a.vc_h;
    kp = reinterpret_cast<const char*>(k + (k0 + lr) * k1 + ch * 8);
    vp = reinterpret_cast<const char*>(v + (k0 + lr) * v1 + ch * 8);
    ks = k1 * (RS * 2);
    vs = v1 * (RS * 2);
  };
  auto fetch = [&](int stage) {
    if (left > 0) {
      char* st = ring + stage * SLAB + tile_at<HD>(lr, ch);
      const bool full = rows >= NK && a.hd == HD;
#pragma unroll
      for (int i = 0; i < NK / RS; ++i) {
        char* d = RS % 8 == 0 ? st + i * RS * HD * 2 : ring + stage * SLAB + tile_at<HD>(lr + i * RS, ch);
        const bool ok = full || (in && lr + i * RS < rows);
        cp_async16(d, ok ? kp + i * ks : (const char*)a.q, ok ? 16 : 0);
        cp_async16(d + NK * HD * 2, ok ? vp + i * vs : (const char*)a.q, ok ? 16 : 0);
      }
      if (--left > 0) {
        if (cur_skip(ahead, a, NK, WARPS) && !fresh && rows > WARPS * NK) {
          kp += ks * (WARPS * NK / RS);
          vp += vs * (WARPS * NK / RS);
          rows -= WARPS * NK;
        } else {
          aim();
        }
      }
    }
    cp_async_commit();
  };
  if (left > 0) {
    cur_skip(ahead, a, NK, warp);
    aim();
  }
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) fetch(i);

  // ---- the units of the share ---------------------------------------------------------------------
  long done = 0, mine = warp;                                   // tiles before this unit, this warp's next
  int stage = 0;
  while (done < share) {
    const int b = cur.b, h = cur.u / a.nrb, rb = cur.u - h * a.nrb, r0 = rb * a.rows;
    const long bh = (long)b * a.nkv + h;
    const int t1 = (int)min((long)cur.n, cur.t + (share - done));
    const int ncache = (cur.len + NK - 1) / NK;
    const long end = done + (t1 - cur.t);
    // B fragments of Q^T: rows r0 + 8 nt + g
    uint32_t qf[NT][HD / 16][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = r0 + 8 * nt + g, tok = div_group(a, row);
      const T* p = (const T*)a.q + b * a.q_b + tok * a.q_t + (long)(h * a.group + row - tok * a.group) * a.q_h;
#pragma unroll
      for (int k = 0; k < HD / 16; ++k)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int d = k * 16 + e * 8 + 2 * t;
          qf[nt][k][e] = row < R && d < a.hd ? *reinterpret_cast<const uint32_t*>(p + d) : 0u;
        }
    }
    float o[HD / 16][NT][4];                                    // channels 16 mt + g (+ 8), rows 8 nt + 2 t (+ 1)
#pragma unroll
    for (int i = 0; i < HD / 16; ++i)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) o[i][nt][0] = o[i][nt][1] = o[i][nt][2] = o[i][nt][3] = 0.f;
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -CUDART_INF_F;
      l[nt][0] = l[nt][1] = 0.f;                                // this lane's keys only, until the end
    }

    for (; mine < end; mine += WARPS) {
      const int tt = cur.t + (int)(mine - done);
      cp_async_wait_group<STAGES - 2>();
      __syncwarp();                                             // the slab is there, the one before it has been read
      fetch(stage == 0 ? STAGES - 1 : stage - 1);
      char* sk = ring + stage * SLAB;
      char* sv = sk + NK * HD * 2;
      const bool tail = tt >= ncache;
      const int k0 = (tail ? tt - ncache : tt) * NK, nk = min(NK, (tail ? a.T : cur.len) - k0);
      // A hidden row's NaN or infinity must not meet its zero probability in the product: what is not finite
      // in V is taken out of the slab, and added by hand, after the product, to the rows that see it.
      bool bad = false;
      if (tail) {
        if (rb == 0) put_slab<T, HD, NK>(sk, a, b, h, cur.len, k0, nk, lane, 32);
        for (int i = lane; i < NK * C; i += 32) bad |= any_inf<T>(*reinterpret_cast<const uint4*>(sv + i * 16));
        bad = __any_sync(0xffffffffu, bad);
        if (bad) {
          __syncwarp();
          for (int i = lane; i < NK * HD; i += 32) {
            unsigned short* p = reinterpret_cast<unsigned short*>(sv + tile_at<HD>(i / HD, (i % HD) >> 3) + (i & 7) * 2);
            if ((*p & Inf<T>::mask) == Inf<T>::mask) *p = 0;
          }
          __syncwarp();
        }
      }
#pragma unroll 1
      for (int kk = 0; kk < NK; kk += 16 * KG) {
        if (kk >= nk) break;
        // S^T of 16 KG keys: rows kk + 16 q + g (+ 8), columns 8 nt + 2 t (+ 1)
        float s[KG][NT][4];
#pragma unroll
        for (int q = 0; q < KG; ++q)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) s[q][nt][0] = s[q][nt][1] = s[q][nt][2] = s[q][nt][3] = 0.f;
#pragma unroll
        for (int k = 0; k < HD / 16; ++k)
#pragma unroll
          for (int q = 0; q < KG; ++q) {
            uint32_t f[4];                                      // A: 16 keys x 16 channels
            ldsm_x4(f[0], f[1], f[2], f[3], sk + tile_at<HD>(kk + 16 * q + (lane & 15), 2 * k + (lane >> 4)));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16<T>(s[q][nt], f, qf[nt][k][0], qf[nt][k][1]);
          }
        if (kk + 16 * KG > nk || tail) {
#pragma unroll
          for (int q = 0; q < KG; ++q)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const int j = kk + 16 * q + g + 8 * x;
              uint32_t vis = j < nk ? ~0u : 0u;
              if (tail) vis &= sees<2 * NT>(a, b, k0 + j, R, [=](int i) { return r0 + (i >> 1) * 8 + 2 * t + (i & 1); });
#pragma unroll
              for (int i = 0; i < 2 * NT; ++i)
                if (!(vis >> i & 1)) s[q][i >> 1][2 * x + (i & 1)] = -CUDART_INF_F;
            }
        }
        if (a.scores) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int row = r0 + 8 * nt + 2 * t + e;
              if (row < R) {
                float* p = a.scores + (bh * R + row) * a.sp + (tail ? cur.len : 0) + k0 + kk + g;
#pragma unroll
                for (int q = 0; q < KG; ++q)
#pragma unroll
                  for (int x = 0; x < 2; ++x)
                    if (kk + 16 * q + g + 8 * x < nk) p[16 * q + 8 * x] = s[q][nt][2 * x + e] * a.scale_log2;
              }
            }
        }
        // does a score pass its row's reference?
        float mx[NT][2];
        bool far = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = fmaxf(s[0][nt][e], s[0][nt][2 + e]);
#pragma unroll
            for (int q = 1; q < KG; ++q) x = fmaxf(x, fmaxf(s[q][nt][e], s[q][nt][2 + e]));
            mx[nt][e] = x;
            far |= (x - m[nt][e]) * a.scale_log2 > Ref<T>::lazy;
          }
        if (__any_sync(0xffffffffu, far)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float x = fmaxf(mx[nt][e], m[nt][e]);
              x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
              x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
              x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
              const float al = x == -CUDART_INF_F ? 1.f : ex2((m[nt][e] - x) * a.scale_log2);
              m[nt][e] = x;
              l[nt][e] *= al;
#pragma unroll
              for (int i = 0; i < HD / 16; ++i) {
                o[i][nt][e] *= al;
                o[i][nt][2 + e] *= al;
              }
            }
        }
        uint32_t pf[KG][NT][2], pr[KG][NT][2];                  // B: 16 keys x 8 rows, and what its rounding left
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float b0 = m[nt][0] == -CUDART_INF_F ? 0.f : m[nt][0], b1 = m[nt][1] == -CUDART_INF_F ? 0.f : m[nt][1];
#pragma unroll
          for (int q = 0; q < KG; ++q)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const float p0 = ex2(fmaf(s[q][nt][2 * x] - b0, a.scale_log2, Ref<T>::up));
              const float p1 = ex2(fmaf(s[q][nt][2 * x + 1] - b1, a.scale_log2, Ref<T>::up));
              l[nt][0] += p0;
              l[nt][1] += p1;
              const uint32_t p = pack2<T>(p0, p1);
              pf[q][nt][x] = transpose8(p);
              pr[q][nt][x] = transpose8(rest2<T>(p0, p1, p));
            }
        }
        // O^T += V^T P^T
#pragma unroll
        for (int i = 0; i < HD / 16; ++i)
#pragma unroll
          for (int q = 0; q < KG; ++q) {
            uint32_t f[4];                                      // A: 16 channels x 16 keys, V read transposed
            ldsm_x4_t(f[0], f[1], f[2], f[3],
                      sv + tile_at<HD>(kk + 16 * q + (lane & 7) + (lane >> 4) * 8, 2 * i + ((lane >> 3) & 1)));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma16<T>(o[i][nt], f, pf[q][nt][0], pf[q][nt][1]);
              mma16<T>(o[i][nt], f, pr[q][nt][0], pr[q][nt][1]);
            }
          }
      }
      if (bad) {
        const T* vn = (const T*)a.vn + b * a.vn_b + h * a.vn_h;
        for (int j = 0; j < nk; ++j) {
          const uint32_t vis = sees<2 * NT>(a, b, k0 + j, R, [=](int i) { return r0 + (i >> 1) * 8 + 2 * t + (i & 1); });
#pragma unroll
          for (int i = 0; i < HD / 8; ++i) {
            if (i * 8 >= a.hd) break;
            const float v = Elem<T>::to(vn[(k0 + j) * a.vn_t + i * 8 + g]);
            if (isfinite(v)) continue;
#pragma unroll
            for (int r = 0; r < 2 * NT; ++r)
              if (vis >> r & 1) o[i >> 1][r >> 1][(i & 1) * 2 + (r & 1)] += v;
          }
        }
      }
      stage = stage == STAGES - 1 ? 0 : stage + 1;
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 4);
        l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 8);
        l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 16);
      }

    // ---- join the warps: 2 and 3 hand over to 0 and 1, then 1 to 0 -------------------------------
    constexpr int MT = HD / 16, PER = MT * NT * 4 * 32;
    float* sM = sJ + 2 * PER;                                 // [2][8 NT][2]
    auto give = [&](int slot) {
      float* buf = sJ + slot * PER + lane;
      float* ml = sM + slot * NT * 16 + 4 * t;                // rows 2 t, 2 t + 1 of a column group
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) buf[((i * NT + nt) * 4 + e) * 32] = o[i][nt][e];
      if (g == 0) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          *reinterpret_cast<float4*>(ml + nt * 16) = make_float4(m[nt][0], l[nt][0], m[nt][1], l[nt][1]);
      }
    };
    auto take = [&](int slot) {
      const float* buf = sJ + slot * PER + lane;
      const float* ml = sM + slot * NT * 16 + 4 * t;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float m2 = ml[nt * 16 + 2 * e], x = fmaxf(m[nt][e], m2);
          const float e0 = x == -CUDART_INF_F ? 1.f : ex2((m[nt][e] - x) * a.scale_log2), e1 = x == -CUDART_INF_F ? 0.f : ex2((m2 - x) * a.scale_log2);
          m[nt][e] = x;
          l[nt][e] = l[nt][e] * e0 + ml[nt * 16 + 2 * e + 1] * e1;
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int y = 0; y < 2; ++y)
              o[i][nt][2 * y + e] = o[i][nt][2 * y + e] * e0 + buf[((i * NT + nt) * 4 + 2 * y + e) * 32] * e1;
        }
    };
    if (warp >= 2) give(warp - 2);
    __syncthreads();
    if (warp < 2) take(warp);
    __syncwarp();
    if (warp == 1) give(1);                                   // only this warp has read slot 1
    __syncthreads();
    if (warp == 0) take(1);
    __syncthreads();                                          // the next unit may end at once for warp 3
    if (warp == 0) {
      const bool first = cur.t == 0, all = first && t1 == cur.n;
      const long slot = 2L * blockIdx.x + (first ? 1 : 0);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int row = r0 + 8 * nt + 2 * t + e;
          if (row >= R) continue;
          if (all) {
            const int tok = div_group(a, row);
            const float inv = l[nt][e] == 0.f ? 0.f : 1.f / l[nt][e];
            T* p = (T*)a.o + (((long)b * a.T + tok) * a.nkv * a.group + h * a.group + row - tok * a.group) * a.hd + g;
#pragma unroll
            for (int i = 0; i < HD / 8; ++i)
              if (i * 8 < a.hd) p[i * 8] = Elem<T>::of(o[i >> 1][nt][(i & 1) * 2 + e] * inv);
            if (a.norm && g == 0) reinterpret_cast<float2*>(a.norm)[bh * R + row] = row_norm(m[nt][e] * a.scale_log2, l[nt][e] * Ref<T>::down);
          } else {
            const long at = slot * a.rows + row - r0;
            float* p = a.part_o + at * a.hd + g;
#pragma unroll
            for (int i = 0; i < HD / 8; ++i)
              if (i * 8 < a.hd) p[i * 8] = o[i >> 1][nt][(i & 1) * 2 + e] * Ref<T>::down;
            if (g == 0) *reinterpret_cast<float2*>(a.part_ml + at * 2) = make_float2(m[nt][e] * a.scale_log2, l[nt][e] * Ref<T>::down);
          }
        }
    }
    done = end;
    cur.t = 0;
    cur_next_unit(cur, a, NK);
  }
}

template <typename T, int HD, int NT>
int run_tc(const KvAttnArgs& a, cudaStream_t st) {
  const size_t sm = std::max<size_t>(WARPS * STAGES * SLAB + join_bytes<HD, NT>(), (size_t)plan_ints(a.B) * 4);
  const cudaError_t e = cudaFuncSetAttribute(kv_attn_tc_k<T, HD, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sm);
  if (e != cudaSuccess) return (int)e;
  kv_attn_tc_k<T, HD, NT><<<a.whole ? a.B * a.nkv * a.nrb : a.ctas, 32 * WARPS, sm, st>>>(a, a.ctas);
  return launched();
}
template <typename T, int HD>
int launch_tc(const KvAttnArgs& a, cudaStream_t st) {
  return a.rows == 8 ? run_tc<T, HD, 1>(a, st) : run_tc<T, HD, 2>(a, st);
}

}  // namespace kv
}  // namespace s0

// Heads of up to 128 channels, a multiple of 8, in a 16-bit type, all rows 16-byte aligned.
bool kv_attn_tc_takes(const KvAttnArgs& a, int dtype) {
  if (dtype == 0 || a.hd > 128 || a.hd % 8) return false;
  for (long s : {a.q_b, a.q_t, a.q_h, a.kn_b, a.kn_t, a.kn_h, a.vn_b, a.vn_t, a.vn_h, a.kc_b, a.kc_h, a.kc_s, a.vc_b, a.vc_h, a.vc_s})
    if (s % 8) return false;
  for (const void* p : {a.q, a.kn, a.vn, (const void*)a.kc, (const void*)a.vc})
    if (reinterpret_cast<uintptr_t>(p) % 16) return false;
  return true;
}

void kv_attn_tc_plan(KvAttnArgs& a, int sms) {
  using namespace s0::kv;
  const int R = a.T * a.group;
  if (R > 16) return kv_attn_t5_plan(a, sms);
  a.tc = 1;
  a.rows = R <= 8 ? 8 : 16;
  a.nrb = 1;
  a.tile = a.hd > 64 ? slab_keys<128>() : slab_keys<64>();
  a.ctas = 2 * sms;
  a.min_per = WARPS;
  a.whole = a.S + a.T <= 4 * a.tile * WARPS;
  a.extra = 8;
  a.least = 16;
}

int kv_attn_tc_launch(const KvAttnArgs& a, int dtype, cudaStream_t st) {
  using namespace s0::kv;
  if (a.tc == 2) return kv_attn_t5_launch(a, dtype, st);
  if (dtype == 1) return a.hd > 64 ? launch_tc<__half, 128>(a, st) : launch_tc<__half, 64>(a, st);
  return a.hd > 64 ? launch_tc<__nv_bfloat16, 128>(a, st) : launch_tc<__nv_bfloat16, 64>(a, st);
}
