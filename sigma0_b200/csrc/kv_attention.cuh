// Shared parts of the cache kernels (kv_attention*.cu, kv_evict.cu): how the
// keys of all sequences are split over the CTAs, and element types.
//
// The lengths live on the device, so the host cannot balance a ragged batch.  Every CTA derives
// the same split from them instead: the key tiles of all units (sequence, key head, block of query
// rows) are laid end to end, and CTA c takes tiles [c per, (c + 1) per).  A unit that one CTA holds
// whole is written out by it; one that several share leaves partial results (unnormalised output,
// running maximum and sum), which a second kernel joins.  A CTA has at most two such pieces: the
// end of one unit (slot 2 c) and the beginning of another (slot 2 c + 1).
//
// A unit costs something of its own (queries, the mask, the new rows, its output), and the trips to
// memory that a unit of few tiles takes are not covered by the streaming of its own tiles: it counts as
// n tiles and `a.extra` more, `a.least` in all at least.  The line is one of these costs; the surplus lies
// at the beginning of a unit, and a CTA whose share begins within it begins with tile 0, so tile t of a unit
// whose costs begin at s is CTA (s + surplus + t) / per's.
// The two numbers come from sweeps of each of the three kernels (tiles of 4 to 128 keys): 14 ragged batches, 16-bit and
// float32, one to 200 rows, contexts of up to 26,000.  Times in us at extra and least 0 and 0 / 8 and 16 / 8 and 20 /
// 24 and 32: one token of 64 books 308 / 294 / 298 / 294, of 40 books of up to 1,500 tokens 69 / 50 / 48 / 50, a tree of 64
// 579 / 368 / 345 / 349, 200 new tokens of 5 books 384 / 97 / 93 / 91, the float32 message 224 / 108 / 103 / 116.  From 8 on
// it is flat: 8 with 16 or 20 serves all.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>
#include <atomic>

#include "common.cuh"
#include "launchers.h"

namespace s0 {
namespace kv {

// kernels launched by these files, in all threads: a call takes one or two, by its sizes
inline std::atomic<long> launches{0};
inline int launched() {
  ++launches;
  return (int)cudaGetLastError();
}

template <typename T> struct Elem;
template <> struct Elem<float> {
  S0_DEV static float to(float x) { return x; }
  S0_DEV static float of(float x) { return x; }
};
template <> struct Elem<__half> {
  S0_DEV static float to(__half x) { return __half2float(x); }
  S0_DEV static __half of(float x) { return __float2half_rn(x); }
};
template <> struct Elem<__nv_bfloat16> {
  S0_DEV static float to(__nv_bfloat16 x) { return __bfloat162float(x); }
  S0_DEV static __nv_bfloat16 of(float x) { return __float2bfloat16_rn(x); }
};

template <typename T> S0_DEV uint32_t pack2(float lo, float hi);
template <> S0_DEV uint32_t pack2<__nv_bfloat16>(float lo, float hi) { return pack_bf16(lo, hi); }
template <> S0_DEV uint32_t pack2<__half>(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// what two probabilities lose when they are packed, packed itself: the pair holds 16 (bf16) or 22 (fp16) bits of each
template <typename T> S0_DEV uint32_t rest2(float lo, float hi, uint32_t packed);
template <> S0_DEV uint32_t rest2<__nv_bfloat16>(float lo, float hi, uint32_t packed) {
  return pack_bf16(lo - __uint_as_float(packed << 16), hi - __uint_as_float(packed & 0xffff0000u));
}
template <> S0_DEV uint32_t rest2<__half>(float lo, float hi, uint32_t packed) {
  const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&packed));
  return pack2<__half>(lo - v.x, hi - v.y);
}
// Probabilities of the tensor-core kernels: 2^((s - m) scale + up), s the products as they come.  m is a score of the row (the
// difference is exact for the scores next to it, however large they are) and moves when one passes it by `lazy` in base 2.
// fp16 keeps nothing below 2^-25, which the many small ones of a long context are beside one large one: 2^11 up that
// is 2^-36 of the largest.
template <typename T> struct Ref;
template <> struct Ref<__nv_bfloat16> { static constexpr float up = 0.f, lazy = 8.f, down = 1.f; };
template <> struct Ref<__half> { static constexpr float up = 11.f, lazy = 4.f, down = 1.f / 2048; };  // down = 2^-up
// exponent bits all ones: infinity or NaN
template <typename T> struct Inf;
template <> struct Inf<__nv_bfloat16> { static constexpr uint32_t mask = 0x7f80u; };
template <> struct Inf<__half> { static constexpr uint32_t mask = 0x7c00u; };
template <typename T> S0_DEV bool any_inf(uint4 x) {
  constexpr uint32_t m = Inf<T>::mask, hi = m << 16;
  auto bad = [](uint32_t v) { return (v & m) == m || (v & hi) == hi; };
  return bad(x.x) || bad(x.y) || bad(x.z) || bad(x.w);
}

// cached tokens of sequence b: a length outside [0, S] cannot be read or written past the cache
S0_DEV int cached(const KvAttnArgs& a, int b) { return min(max(__ldg(a.lengths + b), 0), a.S); }

// key tiles of a sequence: its cached tokens, then the new ones (tiles never mix the two)
S0_DEV int tiles_of(const KvAttnArgs& a, int len, int KT) { return (len + KT - 1) / KT + (a.T + KT - 1) / KT; }

S0_DEV int cost_of(const KvAttnArgs& a, int tiles) { return max(tiles + a.extra, a.least); }

// pre[b] = costs, pre[B + 1 + b] = tiles of one (head, row block) before sequence b; returns all costs.  Called
// by all threads of the block; pre: plan_ints(B) of shared memory.
__host__ __device__ constexpr int plan_ints(int B) { return 2 * (B + 1) + 64; }
S0_DEV long plan_prefix(const KvAttnArgs& a, int KT, int* pre) {
  int *s_w = pre + 2 * (a.B + 1), *tl = pre + a.B + 1;
  const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 31, warp = tid >> 5;
  const int per = (a.B + nt - 1) / nt, b0 = min(a.B, tid * per), b1 = min(a.B, b0 + per);
  int cost = 0, tiles = 0;
  for (int b = b0; b < b1; ++b) {
    const int n = tiles_of(a, cached(a, b), KT);
    cost += cost_of(a, n);
    tiles += n;
  }
  int ic = cost, it = tiles;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, ic, o), y = __shfl_up_sync(0xffffffffu, it, o);
    if (lane >= o) {
      ic += x;
      it += y;
    }
  }
  if (lane == 31) {
    s_w[warp] = ic;
    s_w[32 + warp] = it;
  }
  __syncthreads();
  ic -= cost;
  it -= tiles;
  for (int w = 0; w < warp; ++w) {
    ic += s_w[w];
    it += s_w[32 + w];
  }
  for (int b = b0; b < b1; ++b) {
    pre[b] = ic;
    tl[b] = it;
    const int n = tiles_of(a, cached(a, b), KT);
    ic += cost_of(a, n);
    it += n;
  }
  if (b1 == a.B && b0 < a.B) {
    pre[a.B] = ic;
    tl[a.B] = it;
  }
  __syncthreads();
  return pre[a.B];
}

struct Plan {
  long total;  // costs of all units
  long per;    // costs of a CTA
};
S0_DEV Plan make_plan(const KvAttnArgs& a, long costs, int ctas, int min_per) {
  Plan p;
  p.total = costs * a.nkv * a.nrb;
  p.per = max((long)min_per, (p.total + ctas - 1) / ctas);
  return p;
}

// row / group for rows below 2^20: (row + 1/2) / group is at least 1 / (2 group) away from an integer
S0_DEV int div_group(const KvAttnArgs& a, int row) { return (int)((row + 0.5f) * a.inv_group); }

// Which of CNT rows (row(0), row(1), ...) see new token i, one bit each.  Indices past the end are clamped and
// the choice between a mask and the causal order stands outside, so that the loads are in flight together.
template <int CNT, typename F>
S0_DEV uint32_t sees(const KvAttnArgs& a, int b, int i, int R, F row) {
  uint32_t bits = 0;
  const int j = min(i, a.T - 1);
  if (a.mask) {
    const unsigned char* m = a.mask + b * a.mask_b + j;
    unsigned char x[CNT];
#pragma unroll
    for (int k = 0; k < CNT; ++k) x[k] = m[(long)min(div_group(a, row(k)), a.T - 1) * a.T];
#pragma unroll
    for (int k = 0; k < CNT; ++k) bits |= (uint32_t)((x[k] != 0) & (row(k) < R)) << k;
  } else {
#pragma unroll
    for (int k = 0; k < CNT; ++k) bits |= (uint32_t)((j <= div_group(a, row(k))) & (row(k) < R)) << k;
  }
  return bits;
}

// 2^x: results below 2^-126 become 0
S0_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A unit and the place in it; steps from unit to unit in the plan's order.
struct Cur {
  int b, u, len, n, t;  // sequence, head * nrb + row block, cached tokens, tiles, tile
  int next;             // cached tokens of sequence b + 1: the trip for them is over before they are wanted
};
S0_DEV void cur_set(Cur& c, const KvAttnArgs& a, int KT, int len) {
  c.len = len;
  c.n = tiles_of(a, len, KT);
  c.next = c.b + 1 < a.B ? cached(a, c.b + 1) : 0;
}
S0_DEV void cur_next_unit(Cur& c, const KvAttnArgs& a, int KT) {
  if (++c.u == a.nkv * a.nrb) {
    c.u = 0;
    if (++c.b < a.B) cur_set(c, a, KT, c.next);
  }
}
// true while the unit stays the same
S0_DEV bool cur_skip(Cur& c, const KvAttnArgs& a, int KT, int by) {
  c.t += by;
  if (c.t < c.n) return true;
  while (c.b < a.B && c.t >= c.n) {
    c.t -= c.n;
    cur_next_unit(c, a, KT);
  }
  return false;
}

// The unit and tile at cost w of the line; returns how many tiles lie before it.
S0_DEV long find_tile(Cur& c, const KvAttnArgs& a, const int* s_pre, long w, int KT) {
  const long hr = (long)a.nkv * a.nrb;
  int lo = 0, hi = a.B - 1;
  while (lo < hi) {  // the last b with pre[b] * hr <= w
    const int mid = (lo + hi + 1) >> 1;
    if ((long)s_pre[mid] * hr <= w) lo = mid; else hi = mid - 1;
  }
  const long rem = w - (long)s_pre[lo] * hr;
  const int cost = s_pre[lo + 1] - s_pre[lo];
  c.b = lo;
  cur_set(c, a, KT, cached(a, lo));
  c.u = (int)(rem / cost);
  c.t = max(0, (int)(rem - (long)c.u * cost) - (cost - c.n));
  return (long)s_pre[a.B + 1 + lo] * hr + (long)c.u * c.n + c.t;
}

// The first tile of this CTA and how many it has.  a.whole: one unit per CTA (caches that are short
// enough); otherwise the even split, whose prefix table CTA 0 leaves for the join.
S0_DEV long cta_share(Cur& c, const KvAttnArgs& a, int KT, int* scratch, int ctas) {
  const int hr = a.nkv * a.nrb;
  if (a.whole) {
    c.b = blockIdx.x / hr;
    c.u = blockIdx.x - c.b * hr;
    c.t = 0;
    cur_set(c, a, KT, cached(a, c.b));
    return c.n;
  }
  const Plan p = make_plan(a, plan_prefix(a, KT, scratch), ctas, a.min_per);
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i <= a.B; i += blockDim.x) a.prefix[i] = scratch[i];
  const long w0 = (long)blockIdx.x * p.per, w1 = w0 + p.per;
  if (w0 >= p.total) return 0;
  const long end = w1 < p.total ? find_tile(c, a, scratch, w1, KT) : (long)scratch[2 * a.B + 1] * hr;
  return end - find_tile(c, a, scratch, w0, KT);
}

// Programmatic launch: the kernel behind this one may be set up while it runs, and waits for its results.
S0_DEV void join_may_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
S0_DEV void join_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename... P, typename... A>
int launch_after(void (*k)(P...), unsigned blocks, int threads, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(threads);
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  ++launches;
  return (int)cudaLaunchKernelEx(&cfg, k, P(args)...);
}

// What a row's weights need: p = 2^(s - x) y, (x, y) = (maximum, 1 / sum) and (0, 0) where it saw nothing.  Apart, since a
// sum's logarithm would lose its bits in that of a large maximum.
S0_DEV float2 row_norm(float m, float l) { return make_float2(m == -CUDART_INF_F ? 0.f : m, l == 0.f ? 0.f : 1.f / l); }

}  // namespace kv
}  // namespace s0
