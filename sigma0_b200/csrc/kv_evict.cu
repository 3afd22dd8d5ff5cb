// Which cached tokens stay, and moving their rows: eviction by accumulated attention weight, and
// the acceptance of a drafted tree.
//
// Eviction.  Slot i of a unit (layer, sequence, key head) has the key
//   top            if its position is among the first `sinks` or the last `recent` seen,
//   ord(weight_i)  otherwise (ord: unsigned integers in the order of the floats, NaN above all),
// and the min(len, keep) largest stay, the lower slot first among equals.  The order of cached rows
// means nothing to the attention, so only what lies behind the new end moves: the i-th survivor
// there goes to the i-th free slot before it.  That is at most len - keep rows, where closing the
// gaps in order would move nearly all.
//   evict_select_k   one block per unit: radix select of the threshold (four passes over 8 bits),
//                    then ordered ranks by block scans; writes the metadata and the list of moves;
//   evict_move_k     the rows of all units, 16 bytes a thread where the layout allows.
//
// Acceptance.  The walk down a tree of drafted tokens takes the lowest child whose token is the
// model's token after the node, until there is none; row len + path[j] moves to len + j.  A child
// has a higher index than its parent, so path[j] >= j and rows can move upwards in order.
#include <algorithm>

#include "common.cuh"
#include "launchers.h"

namespace s0 {
namespace kv {

constexpr int ET = 512;

S0_DEV uint32_t order_key(float w, int pos, int seen, const KvEvictArgs& a) {
  if (pos >= seen - a.recent || pos < a.sinks) return 0xffffffffu;
  if (w != w) return 0xfffffffeu;
  const uint32_t u = __float_as_uint(w + 0.f);  // -0 becomes 0
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// exclusive sums of three 0/1 flags of every thread (packed into 21 bits each) and their totals
S0_DEV unsigned long long block_scan(unsigned long long v, unsigned long long* s_w, unsigned long long& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned long long inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long y = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += y;
  }
  __syncthreads();
  if (lane == 31) s_w[warp] = inc;
  __syncthreads();
  unsigned long long base = 0, sum = 0;
  for (int w = 0; w < ET / 32; ++w) {
    if (w < warp) base += s_w[w];
    sum += s_w[w];
  }
  total = sum;
  return base + inc - v;
}

__global__ void __launch_bounds__(ET) evict_select_k(KvEvictArgs a) {
  __shared__ int s_hist[256];
  __shared__ uint32_t s_prefix;
  __shared__ int s_need;
  __shared__ unsigned long long s_w[ET / 32];
  const int tid = threadIdx.x;
  const long u = blockIdx.x;
  const int h = (int)(u % a.nkv), b = (int)(u / a.nkv % a.B), n = (int)(u / a.nkv / a.B);
  const float* w = a.weight + n * a.w_n + b * a.w_b + h * a.w_h;
  const int* p = a.positions + n * a.p_n + b * a.p_b + h * a.p_h;
  float* wo = a.weight_out + n * a.wo_n + b * a.wo_b + h * a.wo_h;
  int* po = a.positions_out + n * a.po_n + b * a.po_b + h * a.po_h;
  const int len = min(max(a.lengths[b], 0), a.S), fin = min(len, a.keep), seen = a.seen[b];
  int2* mv = a.moves + u * a.keep;

  int moved = 0;
  if (len > fin) {
    // the fin-th largest key, 8 bits at a time; s_need: how many of the keys that share the prefix stay
    if (tid == 0) { s_prefix = 0; s_need = fin; }
    for (int sh = 24; sh >= 0; sh -= 8) {
      if (tid < 256) s_hist[tid] = 0;
      __syncthreads();
      const uint32_t prefix = s_prefix, high = sh == 24 ? 0u : 0xffffffffu << (sh + 8);
      for (int i = tid; i < len; i += ET) {
        const uint32_t k = order_key(w[i], p[i], seen, a);
        if ((k & high) == prefix) atomicAdd(&s_hist[(k >> sh) & 255], 1);
      }
      __syncthreads();
      if (tid == 0) {
        int need = s_need, d = 255;
        while (d > 0 && s_hist[d] < need) need -= s_hist[d--];
        s_prefix = prefix | ((uint32_t)d << sh);
        s_need = need;
      }
      __syncthreads();
    }
    const uint32_t thr = s_prefix;
    const int ties = s_need;
    // ordered ranks: equal keys, free slots before the new end, survivors behind it
    int eq0 = 0, hole0 = 0;
    for (int i0 = 0; i0 < len; i0 += ET) {
      const int i = i0 + tid;
      const uint32_t k = i < len ? order_key(w[i], p[i], seen, a) : 0;
      const bool in = i < len, eq = in && k == thr;
      unsigned long long tot;
      const int er = eq0 + (int)block_scan(eq, s_w, tot);
      eq0 += (int)tot;
      const bool stay = in && (k > thr || (eq && er < ties));
      const bool hole = i < fin && !stay, mover = i >= fin && stay;
      const unsigned long long at = block_scan((unsigned long long)hole | ((unsigned long long)mover << 32), s_w, tot);
      if (hole) mv[hole0 + (int)(at & 0xffffffffu)].y = i;
      if (mover) mv[moved + (int)(at >> 32)].x = i;
      hole0 += (int)(tot & 0xffffffffu);
      moved += (int)(tot >> 32);
    }
  }
  if (tid == 0) a.count[u] = moved;
  // metadata: what stays in place, then the moved, then the free slots (read before they are cleared
  // when the outputs are the inputs)
  if (wo != w)
    for (int i = tid; i < fin; i += ET) wo[i] = w[i];
  if (po != p)
    for (int i = tid; i < fin; i += ET) po[i] = p[i];
  __syncthreads();
  for (int j = tid; j < moved; j += ET) {
    const int2 m = mv[j];
    wo[m.y] = w[m.x];
    po[m.y] = p[m.x];
  }
  __syncthreads();
  for (int i = fin + tid; i < a.S; i += ET) {
    wo[i] = 0.f;
    po[i] = -1;
  }
}

// V: the widest type that the rows' addresses and lengths are multiples of
template <typename V>
__global__ void __launch_bounds__(256) evict_move_k(KvEvictArgs a, int parts) {
  const long u = blockIdx.x / parts;
  const int part = (int)(blockIdx.x % parts);
  const int h = (int)(u % a.nkv), b = (int)(u / a.nkv % a.B), n = (int)(u / a.nkv / a.B);
  const int C = a.hd * a.esize / (int)sizeof(V);
  const long count = a.count[u];
  const int2* mv = a.moves + u * a.keep;
  char* kc = (char*)a.kc + (n * a.kc_n + b * a.kc_b + h * a.kc_h) * a.esize;
  char* vc = (char*)a.vc + (n * a.vc_n + b * a.vc_b + h * a.vc_h) * a.esize;
  const long ks = a.kc_s * a.esize, vs = a.vc_s * a.esize;
  for (long i = (long)part * 256 + threadIdx.x; i < count * C; i += 256L * parts) {
    const int2 m = mv[i / C];
    const long c = i % C * (long)sizeof(V);
    const V k = *reinterpret_cast<const V*>(kc + m.x * ks + c), v = *reinterpret_cast<const V*>(vc + m.x * vs + c);
    *reinterpret_cast<V*>(kc + m.y * ks + c) = k;
    *reinterpret_cast<V*>(vc + m.y * vs + c) = v;
  }
  if (u < (long)a.B * a.nkv && h == 0 && part == 0 && threadIdx.x == 0)
    a.lengths_out[b] = min(min(max(a.lengths[b], 0), a.S), a.keep);
}

constexpr int CT = 512, CMAX = 1024;

template <typename V>
__global__ void __launch_bounds__(CT) commit_k(KvCommitArgs a) {
  __shared__ int s_par[CMAX], s_path[CMAX];
  __shared__ long s_tok[CMAX], s_tgt[CMAX];
  __shared__ int s_cnt;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = blockIdx.x % a.B, n = blockIdx.x / a.B;
  for (int i = tid; i < a.T; i += CT) {
    s_par[i] = a.parents[b * a.par_b + i];
    s_tok[i] = a.tokens[(long)b * a.T + i];
    s_tgt[i] = a.targets[(long)b * a.T + i];
  }
  __syncthreads();
  if (warp == 0) {
    int cur = 0, cnt = 1;
    if (lane == 0) s_path[0] = 0;
    while (true) {
      const long want = s_tgt[cur];
      int found = -1;
      for (int i0 = (cur + 1) & ~31; i0 < a.T && found < 0; i0 += 32) {   // nodes above cur only: the walk ends
        const int i = i0 + lane;
        const bool fit = i > cur && i < a.T && s_par[i] == cur && s_tok[i] == want;
        const unsigned any = __ballot_sync(0xffffffffu, fit);
        if (any) found = i0 + __ffs(any) - 1;
      }
      if (found < 0) break;
      if (lane == 0) s_path[cnt] = found;
      ++cnt;
      cur = found;
    }
    if (lane == 0) {
      s_cnt = cnt;
      if (n == 0) {
        a.count[b] = cnt;
        a.next[b] = s_tgt[cur];
      }
    }
  }
  __syncthreads();
  const int cnt = s_cnt, len = min(max(a.lengths[b], 0), a.S);
  if (n == 0)
    for (int i = tid; i < a.T; i += CT) a.path[(long)b * a.T + i] = i < cnt ? s_path[i] : -1;

  // rows: a thread owns one column block of one head's K or V rows and moves them in order, eight loads
  // at a time (a destination never lies behind a later source)
  const int C = a.hd * a.esize / (int)sizeof(V);
  const int fit = min(a.T, a.S - len);                   // new rows that are in the cache at all
  for (int i = tid; i < 2 * a.nkv * C; i += CT) {
    const int kv = i / (a.nkv * C), h = i / C % a.nkv;
    const long c = (long)(i % C) * sizeof(V);
    const long rs = (kv ? a.vc_s : a.kc_s) * a.esize;
    char* base = kv ? (char*)a.vc + (n * a.vc_n + b * a.vc_b + h * a.vc_h) * a.esize
                    : (char*)a.kc + (n * a.kc_n + b * a.kc_b + h * a.kc_h) * a.esize;
    base += len * rs + c;
    for (int j0 = 1; j0 < cnt; j0 += 8) {
      V x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j0 + j < cnt && s_path[j0 + j] < fit) x[j] = *reinterpret_cast<const V*>(base + s_path[j0 + j] * rs);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j0 + j < cnt && s_path[j0 + j] < fit) *reinterpret_cast<V*>(base + (j0 + j) * rs) = x[j];
    }
  }
  for (int h = warp; h < a.nkv; h += CT / 32) {
    float* wt = a.weight ? a.weight + n * a.w_n + b * a.w_b + h * a.w_h + len : nullptr;
    int* ps = a.positions ? a.positions + n * a.p_n + b * a.p_b + h * a.p_h + len : nullptr;
    for (int j0 = 0; j0 < fit; j0 += 32) {
      const int j = j0 + lane;
      const bool on = j < cnt && j < fit && s_path[j] < fit;
      const float x = wt && on ? wt[s_path[j]] : 0.f;
      __syncwarp();
      if (j < fit) {
        if (wt) wt[j] = x;
        if (ps) ps[j] = on ? a.seen[b] + j : -1;
      }
      __syncwarp();
    }
  }
}

// the widest access that divides every stride, the row length and the base address
int width_of(int hd, int es, std::initializer_list<long> strides, std::initializer_list<const void*> bases) {
  for (int v = 16; v > es; v >>= 1) {
    bool ok = (hd * es) % v == 0;
    for (long s : strides) ok = ok && (s * es) % v == 0;
    for (const void* p : bases) ok = ok && reinterpret_cast<uintptr_t>(p) % v == 0;
    if (ok) return v;
  }
  return es;
}

}  // namespace kv
}  // namespace s0

int kv_evict_launch(const KvEvictArgs& a, cudaStream_t st) {
  using namespace s0::kv;
  const long units = (long)a.N * a.B * a.nkv;
  if (units <= 0) return 0;
  evict_select_k<<<(unsigned)units, ET, 0, st>>>(a);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return (int)e;
  const int v = width_of(a.hd, a.esize, {a.kc_n, a.kc_b, a.kc_h, a.kc_s, a.vc_n, a.vc_b, a.vc_h, a.vc_s}, {a.kc, a.vc});
  const int parts = (int)std::max<long>(1, std::min<long>(16, (8L * a.sms + units - 1) / units));
  const unsigned grid = (unsigned)(units * parts);
  if (v == 16) evict_move_k<uint4><<<grid, 256, 0, st>>>(a, parts);
  else if (v == 8) evict_move_k<uint2><<<grid, 256, 0, st>>>(a, parts);
  else if (v == 4) evict_move_k<uint32_t><<<grid, 256, 0, st>>>(a, parts);
  else evict_move_k<uint16_t><<<grid, 256, 0, st>>>(a, parts);
  return (int)cudaGetLastError();
}

int kv_commit_launch(const KvCommitArgs& a, cudaStream_t st) {
  using namespace s0::kv;
  const long blocks = (long)a.N * a.B;
  if (blocks <= 0 || a.T <= 0) return 0;
  const int v = width_of(a.hd, a.esize, {a.kc_n, a.kc_b, a.kc_h, a.kc_s, a.vc_n, a.vc_b, a.vc_h, a.vc_s}, {a.kc, a.vc});
  if (v == 16) commit_k<uint4><<<(unsigned)blocks, CT, 0, st>>>(a);
  else if (v == 8) commit_k<uint2><<<(unsigned)blocks, CT, 0, st>>>(a);
  else if (v == 4) commit_k<uint32_t><<<(unsigned)blocks, CT, 0, st>>>(a);
  else commit_k<uint16_t><<<(unsigned)blocks, CT, 0, st>>>(a);
  return (int)cudaGetLastError();
}
