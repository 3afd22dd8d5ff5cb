// Attention of a few new tokens over a key / value cache: the kernel for any element type, head
// size and alignment, and the kernel that joins the pieces of a split (kv_attention_tc.cu has the
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

constexpr int GT = 128;  // threads of the general kernel
constexpr int GK = 32;   // keys of a tile: one per lane in the softmax
constexpr int GR = 8;    // query rows of a block: two per warp
constexpr int GC = 4;    // output columns of a thread: heads up to GT * GC wide

// The general kernel: everything in fp32, one K (then V) tile in shared memory at a time; element
// loads, so any stride and alignment will do.
template <typename T>
__global__ void __launch_bounds__(GT) kv_attn_any_k(KvAttnArgs a) {
  extern __shared__ __align__(16) unsigned char smem[];
  const int hd = a.hd, ldk = hd | 1;           // odd row stride: lanes read 32 rows at one column
  float* sQ = reinterpret_cast<float*>(smem);  // [GR][hd]
  float* sT = sQ + GR * hd;                    // [GK][ldk]
  float* sP = sT + GK * ldk;                   // [GR][GK]
  float* sA = sP + GR * GK;                    // [GR] rescale, then 1 / sum
  uint32_t* sV = reinterpret_cast<uint32_t*>(sA + GR);  // [GR] visible keys of the tile
  int* s_pre = reinterpret_cast<int*>(sV + GR);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int R = a.T * a.group;
  join_may_start();
  const Plan plan = make_plan(a, plan_prefix(a, GK, s_pre), gridDim.x, a.min_per);
  if (blockIdx.x == 0)
    for (int i = tid; i <= a.B; i += GT) a.prefix[i] = s_pre[i];
  long w = blockIdx.x * plan.per;
  const long wend = min(plan.total, w + plan.per);

  while (w < wend) {
    const Seg sg = find_seg(a, s_pre, w, GK);
    const int t1 = (int)min((long)sg.n, sg.t0 + (wend - w));
    const int b = sg.b, h = sg.h, r0 = sg.rb * GR, nr = min(GR, R - r0);
    const int ncache = (sg.len + GK - 1) / GK;
    T* kc = (T*)a.kc + b * a.kc_b + h * a.kc_h;
    T* vc = (T*)a.vc + b * a.vc_b + h * a.vc_h;
    const T* kn = (const T*)a.kn + b * a.kn_b + h * a.kn_h;
    const T* vn = (const T*)a.vn + b * a.vn_b + h * a.vn_h;
    for (int i = tid; i < GR * hd; i += GT) {
      const int r = i / hd, d = i - r * hd;
      float x = 0.f;
      if (r < nr) {
        const int row = r0 + r, t = row / a.group, g = row - t * a.group;
        x = Elem<T>::to(((const T*)a.q)[b * a.q_b + t * a.q_t + (h * a.group + g) * a.q_h + d]) * a.scale_log2;
      }
      sQ[i] = x;
    }
    float acc[GC][GR];
#pragma unroll
    for (int c = 0; c < GC; ++c)
#pragma unroll
      for (int r = 0; r < GR; ++r) acc[c][r] = 0.f;
    float m[2] = {-CUDART_INF_F, -CUDART_INF_F}, l[2] = {0.f, 0.f};  // rows 2 warp, 2 warp + 1

    for (int tt = sg.t0; tt < t1; ++tt) {
      const bool tail = tt >= ncache;
      const int k0 = (tail ? tt - ncache : tt) * GK, lim = tail ? a.T : sg.len;
      const int nk = min(GK, lim - k0);
      const bool put = tail && sg.rb == 0;
      auto load = [&](T* cache, long cs, const T* fresh, long fs) {
        for (int i = tid; i < GK * hd; i += GT) {
          const int j = i / hd, d = i - j * hd;
          T x = Elem<T>::of(0.f);                       // a key past the end contributes 0 * 0
          if (j < nk) {
            x = tail ? fresh[(k0 + j) * fs + d] : cache[(k0 + j) * cs + d];
            if (put && sg.len + k0 + j < a.S) cache[(long)(sg.len + k0 + j) * cs + d] = x;
          }
          sT[j * ldk + d] = Elem<T>::to(x);
        }
      };
      __syncthreads();
      load(kc, a.kc_s, kn, a.kn_t);
      __syncthreads();
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int r = 2 * warp + q, row = r0 + r;
        float s0 = 0.f, s1 = 0.f;
        const float *qr = sQ + r * hd, *kr = sT + lane * ldk;
        int d = 0;
        for (; d + 1 < hd; d += 2) {
          s0 = fmaf(qr[d], kr[d], s0);
          s1 = fmaf(qr[d + 1], kr[d + 1], s1);
        }
        if (d < hd) s0 = fmaf(qr[d], kr[d], s0);
        float s = s0 + s1;
        const bool vis = lane < nk && r < nr && (!tail || sees(a, b, row / a.group, k0 + lane));
        if (!vis) s = -CUDART_INF_F;
        const uint32_t seen = __ballot_sync(0xffffffffu, vis);
        if (a.scores && lane < nk && r < nr)
          a.scores[(((long)b * a.nkv + h) * R + row) * a.sp + (tail ? sg.len : 0) + k0 + lane] = s;
        float mx = s;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        mx = fmaxf(mx, m[q]);
        const float base = mx == -CUDART_INF_F ? 0.f : mx;
        const float al = exp2f(m[q] - base), p = exp2f(s - base);
        m[q] = mx;
        l[q] = l[q] * al + warp_sum(p);
        sP[r * GK + lane] = p;
        if (lane == 0) {
          sA[r] = al;
          sV[r] = seen;
        }
      }
      __syncthreads();
      load(vc, a.vc_s, vn, a.vn_t);
      __syncthreads();
#pragma unroll
      for (int r = 0; r < GR; ++r) {
        const float al = sA[r];
#pragma unroll
        for (int c = 0; c < GC; ++c) acc[c][r] *= al;
      }
      for (int j = 0; j < nk; ++j) {
        float v[GC];
#pragma unroll
        for (int c = 0; c < GC; ++c) v[c] = tid + c * GT < hd ? sT[j * ldk + tid + c * GT] : 0.f;
#pragma unroll
        for (int r = 0; r < GR; ++r) {
          const float p = sP[r * GK + j];
#pragma unroll
          for (int c = 0; c < GC; ++c)
            if (!tail || (sV[r] >> j & 1)) acc[c][r] = fmaf(p, v[c], acc[c][r]);  // 0 times a hidden infinity stays out
        }
      }
      if (put && a.positions && tid < nk && sg.len + k0 + tid < a.S)
        a.positions[b * a.pos_b + h * a.pos_h + sg.len + k0 + tid] = a.seen[b] + k0 + tid;
    }

    const bool first = sg.t0 == 0, last = t1 == sg.n;
    const long slot = 2L * blockIdx.x + (first ? 1 : 0);
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int r = 2 * warp + q;
      if (lane == 0) {
        if (first && last) {
          sA[r] = l[q] == 0.f ? 0.f : 1.f / l[q];
          if (a.lse && r < nr) a.lse[((long)b * a.nkv + h) * R + r0 + r] = lse2(m[q], l[q]);
        } else {
          a.part_ml[(slot * a.rows + r) * 2] = m[q];
          a.part_ml[(slot * a.rows + r) * 2 + 1] = l[q];
        }
      }
    }
    __syncthreads();
    for (int r = 0; r < nr; ++r) {
      const int row = r0 + r, t = row / a.group, g = row - t * a.group;
#pragma unroll
      for (int c = 0; c < GC; ++c) {
        const int d = tid + c * GT;
        if (d >= hd) continue;
        if (first && last)
          ((T*)a.o)[(((long)b * a.T + t) * a.nkv * a.group + h * a.group + g) * hd + d] = Elem<T>::of(acc[c][r] * sA[r]);
        else
          a.part_o[(slot * a.rows + r) * hd + d] = acc[c][r];
      }
    }
    __syncthreads();
    w += t1 - sg.t0;
  }
}

// Joins the pieces of the units that several CTAs share, and adds up the weights.  Blocks
// [0, B heads T): one row's output; the others: JW slots of one (sequence, key head) each.
constexpr int JT = 256, JW = 2048;

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
template <typename T, int WPR>
__global__ void __launch_bounds__(JT) kv_join_k(KvAttnArgs a, int row_blocks) {
  constexpr int RPB = JT / 32 / WPR, COLS = 4;     // rows of a block, columns of a lane at a time
  __shared__ float s_x[JT * COLS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, R = a.T * a.group;
  const bool out = blockIdx.x < (unsigned)row_blocks;
  const int wb = blockIdx.x - row_blocks, nch = (a.S + a.T + JW - 1) / JW;
  const long total = (long)a.B * a.nkv * R, idx = (long)blockIdx.x * RPB + warp / WPR;
  const long bh = out ? min(idx, total - 1) / R : wb / nch;
  const int b = (int)(bh / a.nkv), h = (int)(bh - (long)b * a.nkv);
  join_wait();
  Plan plan{0, 1};
  int n = 1;
  long ub = 0;                                      // first tile of row block 0
  if (!a.whole) {
    plan = make_plan(a, a.prefix[a.B], a.ctas, a.min_per);
    const int p0 = a.prefix[b];
    n = a.prefix[b + 1] - p0;
    ub = (long)p0 * a.nkv * a.nrb + (long)h * a.nrb * n;
  }
  auto pieces = [&](int rb) {
    const long s = ub + (long)rb * n;
    return Pieces{s / plan.per, (s + n - 1) / plan.per};
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
  const int hi = min(a.S, cached(a, b) + a.T), j0 = (wb - (int)bh * nch) * JW;
  if (j0 >= hi) return;
  float add[JW / JT] = {};
  for (int q0 = 0; q0 < R; q0 += JT) {
    __syncthreads();
    for (int q = warp; q < min(JT, R - q0); q += JT / 32) {
      const int row = q0 + q, rb = row / a.rows;
      const Pieces p = pieces(rb);
      float x;
      if (p.c0 == p.c1) {
        x = a.lse[bh * R + row];
      } else {
        float M, L;
        row_sum(a, p, row - rb * a.rows, M, L);
        x = lse2(M, L);
      }
      if (lane == 0) s_x[q] = x;
    }
    __syncthreads();
    for (int q = 0; q < min(JT, R - q0); ++q) {
      const float* sc = a.scores + (bh * R + q0 + q) * a.sp + j0;
      const float ls = s_x[q];
#pragma unroll
      for (int i = 0; i < JW / JT; ++i)
        if (j0 + i * JT + tid < hi) add[i] += ex2(sc[i * JT + tid] - ls);
    }
  }
  float* wt = a.weight + b * a.wt_b + h * a.wt_h + j0;
#pragma unroll
  for (int i = 0; i < JW / JT; ++i)
    if (j0 + i * JT + tid < hi) wt[i * JT + tid] += add[i];
}

template <typename T>
int launch(const KvAttnArgs& a, cudaStream_t st) {
  const size_t sm = (size_t)(GR * a.hd + GK * (a.hd | 1) + GR * GK + 2 * GR) * 4 + (size_t)(a.B + 33) * 4;
  const cudaError_t e = cudaFuncSetAttribute(kv_attn_any_k<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sm);
  if (e != cudaSuccess) return (int)e;
  kv_attn_any_k<T><<<a.ctas, GT, sm, st>>>(a);
  return (int)cudaGetLastError();
}

template <typename T>
int join(const KvAttnArgs& a, cudaStream_t st) {
  // few rows leave room for a block each, whose warps take turns at the pieces
  const long rows = a.whole ? 0 : (long)a.B * a.nkv * a.T * a.group;
  const bool wide = rows > 4L * a.ctas;
  const long row_blocks = wide ? (rows + JT / 32 - 1) / (JT / 32) : rows;
  const long blocks = row_blocks + (a.weight ? (long)a.B * a.nkv * ((a.S + a.T + JW - 1) / JW) : 0);
  if (blocks == 0) return 0;                        // one CTA per unit and no weights: nothing is left to do
  return wide ? launch_after(kv_join_k<T, 1>, (unsigned)blocks, JT, st, a, (int)row_blocks)
              : launch_after(kv_join_k<T, JT / 32>, (unsigned)blocks, JT, st, a, (int)row_blocks);
}

}  // namespace kv
}  // namespace s0

void kv_attn_plan(KvAttnArgs& a, int dtype, int sms) {
  a.tc = kv_attn_tc_takes(a, dtype);
  if (a.tc) return kv_attn_tc_plan(a, sms);
  const size_t sm = (size_t)(s0::kv::GR * a.hd + s0::kv::GK * (a.hd | 1) + s0::kv::GR * s0::kv::GK) * 4;
  const int R = a.T * a.group;
  a.rows = s0::kv::GR;
  a.nrb = (R + a.rows - 1) / a.rows;
  a.tile = s0::kv::GK;
  a.min_per = 4;
  a.whole = 0;
  a.ctas = sms * (int)std::max<size_t>(1, std::min<size_t>(8, (size_t)200 * 1024 / sm));
}

int kv_attn_launch(const KvAttnArgs& a, int dtype, cudaStream_t st) {
  if (a.B <= 0 || a.T <= 0) return 0;
  using namespace s0::kv;
  const int rc = a.tc ? kv_attn_tc_launch(a, dtype, st)
                 : dtype == 0 ? launch<float>(a, st) : dtype == 1 ? launch<__half>(a, st) : launch<__nv_bfloat16>(a, st);
  if (rc) return rc;
  return dtype == 0 ? join<float>(a, st) : dtype == 1 ? join<__half>(a, st) : join<__nv_bfloat16>(a, st);
}
