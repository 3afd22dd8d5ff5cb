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
  const Plan plan = make_plan(a, plan_prefix(a, GK, s_pre), gridDim.x, a.min_per);
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
// [0, units): the output of one unit; the others: 1024 slots of one (sequence, key head) each.
constexpr int JT = 256, JW = 1024;

template <typename T>
__global__ void __launch_bounds__(JT) kv_join_k(KvAttnArgs a, int KT, int ctas) {
  extern __shared__ __align__(16) unsigned char smem[];
  int* s_pre = reinterpret_cast<int*>(smem);
  __shared__ float s_lse[JT];
  const int tid = threadIdx.x, R = a.T * a.group;
  const Plan plan = make_plan(a, plan_prefix(a, KT, s_pre), ctas, a.min_per);
  const long units = (long)a.B * a.nkv * a.nrb;
  const bool out = blockIdx.x < units;
  const long wb = blockIdx.x - units;
  const int nch = (a.S + a.T + JW - 1) / JW;
  const long bh = out ? (long)blockIdx.x / a.nrb : wb / nch;
  const int b = (int)(bh / a.nkv), h = (int)(bh % a.nkv);
  const int n = s_pre[b + 1] - s_pre[b];
  const long ub = (long)s_pre[b] * a.nkv * a.nrb + (long)h * a.nrb * n;   // first tile of row block 0
  // piece i of row block rb: CTA c0 + i
  auto slot_of = [](long c, long c0) { return 2 * c + (c == c0 ? 1 : 0); };

  if (out) {
    const int rb = (int)(blockIdx.x % a.nrb), r0 = rb * a.rows, nr = min(a.rows, R - r0);
    const long s = ub + (long)rb * n, c0 = s / plan.per, c1 = (s + n - 1) / plan.per;
    if (c0 == c1) return;
    for (int i = tid; i < nr * a.hd; i += JT) {
      const int r = i / a.hd, d = i - r * a.hd;
      float M = -CUDART_INF_F, L = 0.f, x = 0.f;
      for (long c = c0; c <= c1; ++c) {
        const long slot = slot_of(c, c0) * a.rows + r;
        const float mi = a.part_ml[slot * 2], li = a.part_ml[slot * 2 + 1], mn = fmaxf(M, mi);
        const float base = mn == -CUDART_INF_F ? 0.f : mn, e0 = exp2f(M - base), e1 = exp2f(mi - base);
        L = L * e0 + li * e1;
        x = x * e0 + a.part_o[slot * a.hd + d] * e1;
        M = mn;
      }
      const int row = r0 + r, t = row / a.group, g = row - t * a.group;
      ((T*)a.o)[(((long)b * a.T + t) * a.nkv * a.group + h * a.group + g) * a.hd + d] =
          Elem<T>::of(L == 0.f ? 0.f : x / L);
    }
    return;
  }
  const int len = cached(a, b), hi = min(a.S, len + a.T), j0 = (int)(wb % nch) * JW;
  if (j0 >= hi) return;
  float add[JW / JT] = {};
  for (int q0 = 0; q0 < R; q0 += JT) {
    const int row = q0 + tid;
    __syncthreads();
    if (row < R) {
      const int rb = row / a.rows, r = row - rb * a.rows;
      const long s = ub + (long)rb * n, c0 = s / plan.per, c1 = (s + n - 1) / plan.per;
      if (c0 == c1) {
        s_lse[tid] = a.lse[bh * R + row];
      } else {
        float M = -CUDART_INF_F, L = 0.f;
        for (long c = c0; c <= c1; ++c) {
          const long slot = slot_of(c, c0) * a.rows + r;
          const float mi = a.part_ml[slot * 2], li = a.part_ml[slot * 2 + 1], mn = fmaxf(M, mi);
          const float base = mn == -CUDART_INF_F ? 0.f : mn;
          L = L * exp2f(M - base) + li * exp2f(mi - base);
          M = mn;
        }
        s_lse[tid] = lse2(M, L);
      }
    }
    __syncthreads();
    for (int q = 0; q < min(JT, R - q0); ++q) {
      const float* sc = a.scores + (bh * R + q0 + q) * a.sp + j0;
      const float ls = s_lse[q];
#pragma unroll
      for (int i = 0; i < JW / JT; ++i)
        if (j0 + i * JT + tid < hi) add[i] += exp2f(sc[i * JT + tid] - ls);
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
  const long units = (long)a.B * a.nkv * a.nrb;
  const long wblocks = a.weight ? (long)a.B * a.nkv * ((a.S + a.T + JW - 1) / JW) : 0;
  kv_join_k<T><<<(unsigned)(units + wblocks), JT, (size_t)(a.B + 33) * 4, st>>>(a, a.tile, a.ctas);
  return (int)cudaGetLastError();
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
