// Which cached tokens stay, and moving their rows: eviction by accumulated attention weight, and
// the acceptance of a drafted tree.
//
// Eviction.  Slot i of a unit (layer, sequence, key head) has the key
//   top            if its position is among the first `sinks` or the last `recent` seen (-1, no position, is in neither),
//   ord(weight_i)  otherwise (ord: unsigned integers in the order of the floats, NaN above all),
// and the min(len, keep) largest stay, the lower slot first among equals.  The order of cached rows
// means nothing to the attention, so only what lies behind the new end moves: the i-th survivor
// there goes to the i-th free slot before it.  That is at most len - keep rows, where closing the
// gaps in order would move nearly all.
// One block per unit: the keys go to shared memory (as far as they fit; beyond that they are formed
// again on every pass), a radix select over 11 + 11 + 10 bits finds the threshold, block scans the ordered
// ranks, and the block moves its own rows, so that the selection of some units runs under the traffic of
// others.  What bounds it is that traffic: 8 bytes read and written per slot and the moved rows.  With
// fewer units than SMs a second kernel moves the rows instead, with several blocks per unit.  Measured: 11,000 -> 2,048
// slots in 4 layers x 16 books x 16 heads of 64: 206 us, 70% of the copy rate; 4,118 -> 4,096 in 24 layers: 183 us (1,147
// with serial digit searches and a scan per 512 slots), bound by the selection: 53% of the issue slots and its barriers.
//
// Acceptance.  The walk down a tree of drafted tokens takes the lowest child whose token is the
// model's token after the node, until there is none; row len + path[j] moves to len + j.  Nodes whose rows lie past
// the last slot were not stored, and the walk does not go to them.  A child
// has a higher index than its parent, so path[j] >= j and rows can move upwards in order.  64 nodes, 24 layers x 32 books: 14.7 us, a chain of three
// trips to memory (tree and lengths, rows, weights); the rows themselves are 5 us.
#include <algorithm>

#include "kv_attention.cuh"

namespace s0 {
namespace kv {

constexpr int EB = 2048;                 // bins of a pass of 11 bits
constexpr uint32_t HELD = 0xffffffffu;   // stays whatever its weight

S0_DEV uint32_t order_key(float w, int pos, int seen, const KvEvictArgs& a) {
  if (pos >= 0 && (pos >= seen - a.recent || pos < a.sinks)) return HELD;
  if (w != w) return 0xfffffffeu;
  const uint32_t u = __float_as_uint(w + 0.f);  // -0 becomes 0
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// exclusive sum over the block and the total; s_w: one value per warp and one more
template <int NT, typename V>
S0_DEV V block_scan(V v, V* s_w, V& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  V inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V y = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += y;
  }
  __syncthreads();
  if (lane == 31) s_w[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    V x = lane < NT / 32 ? s_w[lane] : V(0), y = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const V z = __shfl_up_sync(0xffffffffu, y, o);
      if (lane >= o) y += z;
    }
    if (lane < NT / 32) s_w[lane] = y - x;
    if (lane == NT / 32 - 1) s_w[NT / 32] = y;
  }
  __syncthreads();
  total = s_w[NT / 32];
  return s_w[warp] + inc - v;
}

// the rows of one unit's moves; V: the widest type that the rows' addresses and lengths are multiples of
template <typename V, int U>             // U: pairs of rows in flight per thread
S0_DEV void move_rows(const KvEvictArgs& a, const int2* mv, long u, int count, int i0, int step) {
  const int h = (int)(u % a.nkv), b = (int)(u / a.nkv % a.B), n = (int)(u / a.nkv / a.B);
  const unsigned C = a.hd * a.esize / (int)sizeof(V), total = count * C;
  char* kc = (char*)a.kc + (n * a.kc_n + b * a.kc_b + h * a.kc_h) * a.esize;
  char* vc = (char*)a.vc + (n * a.vc_n + b * a.vc_b + h * a.vc_h) * a.esize;
  const long ks = a.kc_s * a.esize, vs = a.vc_s * a.esize;
  for (unsigned i = i0; i < total; i += U * step) {
    V k[U], v[U];
    int to[U];
#pragma unroll
    for (int x = 0; x < U; ++x) {
      const unsigned j = i + x * step;
      if (j < total) {
        const unsigned r = j / C;
        const int2 m = mv[r];
        const long c = (long)(j - r * C) * sizeof(V);
        k[x] = *reinterpret_cast<const V*>(kc + m.x * ks + c);
        v[x] = *reinterpret_cast<const V*>(vc + m.x * vs + c);
        to[x] = m.y;
      }
    }
#pragma unroll
    for (int x = 0; x < U; ++x) {
      const unsigned j = i + x * step;
      if (j < total) {
        const long c = (long)(j % C) * sizeof(V);
        *reinterpret_cast<V*>(kc + to[x] * ks + c) = k[x];
        *reinterpret_cast<V*>(vc + to[x] * vs + c) = v[x];
      }
    }
  }
}
template <int U>
S0_DEV void move_rows(const KvEvictArgs& a, const int2* mv, long u, int count, int i0, int step) {
  if (a.width == 16) move_rows<uint4, U>(a, mv, u, count, i0, step);
  else if (a.width == 8) move_rows<uint2, U>(a, mv, u, count, i0, step);
  else if (a.width == 4) move_rows<uint32_t, U>(a, mv, u, count, i0, step);
  else move_rows<uint16_t, U>(a, mv, u, count, i0, step);
}

// The digit that holds the need-th largest value of a histogram: its bin, how many of it are needed.
template <int NT>
S0_DEV void find_digit(const int* hist, int need, int* s_w, int* s_found) {
  constexpr int PER = EB / NT;
  const int tid = threadIdx.x, top = EB - 1 - tid * PER;
  int sum = 0, tot;
#pragma unroll
  for (int k = 0; k < PER; ++k) sum += hist[top - k];
  int above = block_scan<NT, int>(sum, s_w, tot);
  if (above < need && need <= above + sum) {
    int k = top;
    while (above + hist[k] < need) above += hist[k--];
    s_found[0] = k;
    s_found[1] = need - above;
    s_found[2] = hist[k];
  }
  __syncthreads();
}

// KEYS: all keys fit into shared memory
template <int NT, bool KEYS>
__global__ void __launch_bounds__(NT, NT == 256 ? 8 : 1536 / NT) evict_k(KvEvictArgs a, int moves_here) {
  extern __shared__ __align__(16) uint32_t s_key[];    // [S], later the list of moves
  __shared__ int s_hist[EB], s_w[NT / 32 + 1], s_found[3];
  __shared__ unsigned long long s_w2[NT / 32 + 1];
  join_may_start();
  const int tid = threadIdx.x;
  const long u = blockIdx.x;
  const int h = (int)(u % a.nkv), b = (int)(u / a.nkv % a.B), n = (int)(u / a.nkv / a.B);
  const float* w = a.weight + n * a.w_n + b * a.w_b + h * a.w_h;
  const int* p = a.positions + n * a.p_n + b * a.p_b + h * a.p_h;
  float* wo = a.weight_out + n * a.wo_n + b * a.wo_b + h * a.wo_h;
  int* po = a.positions_out + n * a.po_n + b * a.po_b + h * a.po_h;
  const int len = min(max(a.lengths[b], 0), a.S), fin = min(len, a.keep), seen = a.seen[b];
  int2* mv = a.moves + u * a.keep;
  const bool cut = len > fin, copy_w = wo != w, copy_p = po != p;
  for (int i = tid; i < EB; i += NT) s_hist[i] = 0;
  __syncthreads();

  // keys, the first histogram, and what stays in place (free slots are overwritten later)
  int held = 0;
#pragma unroll 4
  for (int i = tid; i < a.S; i += NT) {
    const bool in = i < len;
    const float x = in ? w[i] : 0.f;
    const int y = in ? p[i] : -1;
    if (cut && in) {
      const uint32_t k = order_key(x, y, seen, a);
      if (KEYS) s_key[i] = k;
      if (k == HELD) ++held;
      else atomicAdd(&s_hist[k >> 21], 1);
    }
    if (copy_w) wo[i] = i < fin ? x : 0.f;
    if (copy_p) po[i] = i < fin ? y : -1;
  }
  int moved = 0;
  if (cut) {
    auto key = [&](int i) { return KEYS ? s_key[i] : order_key(w[i], p[i], seen, a); };
    int all_held;
    block_scan<NT, int>(held, s_w, all_held);
    uint32_t thr = HELD;
    int ties = fin, equal = all_held;
    if (all_held < fin) {
      find_digit<NT>(s_hist, fin - all_held, s_w, s_found);
      uint32_t prefix = (uint32_t)s_found[0];
      int need = s_found[1];
#pragma unroll
      for (int pass = 1; pass < 3; ++pass) {
        const int sh = pass == 1 ? 10 : 0, bits = pass == 1 ? 11 : 10, above = sh + bits;
        for (int i = tid; i < EB; i += NT) s_hist[i] = 0;
        __syncthreads();
        for (int i = tid; i < len; i += NT) {
          const uint32_t k = key(i);
          if (k >> above == prefix && k != HELD) atomicAdd(&s_hist[(k >> sh) & ((1u << bits) - 1)], 1);
        }
        __syncthreads();
        find_digit<NT>(s_hist, need, s_w, s_found);
        prefix = prefix << bits | (uint32_t)s_found[0];
        need = s_found[1];
      }
      thr = prefix;
      ties = need;
      equal = s_found[2];
    }
    // Ordered ranks: every thread takes a run of slots (an odd number of them, so that the threads of a warp
    // read different banks).  Equal keys first, if not all of them stay; then free slots before the new
    // end and survivors behind it.
    const int run = (len + NT - 1) / NT | 1, i0 = min(len, tid * run), i1 = min(len, i0 + run);
    int rank = 0;
    if (equal != ties) {
      int e = 0, tot;
      for (int i = i0; i < i1; ++i) e += key(i) == thr;
      rank = block_scan<NT, int>(e, s_w, tot);
    }
    // 64 slots of a run at a time: which of them are free, which move
    auto flags = [&](int s0, unsigned long long& holes, unsigned long long& movers) {
      holes = movers = 0;
      for (int i = s0; i < min(i1, s0 + 64); ++i) {
        const uint32_t k = key(i);
        const bool stay = k > thr || (k == thr && rank++ < ties);
        if (i < fin && !stay) holes |= 1ull << (i - s0);
        if (i >= fin && stay) movers |= 1ull << (i - s0);
      }
    };
    const int rank0 = rank;
    unsigned long long holes = 0, movers = 0, mine = 0, tot2;
    for (int s0 = i0; s0 < i1; s0 += 64) {
      flags(s0, holes, movers);
      mine += (unsigned long long)__popcll(holes) | (unsigned long long)__popcll(movers) << 32;
    }
    const unsigned long long at = block_scan<NT, unsigned long long>(mine, s_w2, tot2);
    int hole = (int)(at & 0xffffffffu), mover = (int)(at >> 32);
    moved = (int)(tot2 >> 32);
    rank = rank0;
    for (int s0 = i0; s0 < i1; s0 += 64) {
      if (i1 - i0 > 64) flags(s0, holes, movers);
      for (; holes; holes &= holes - 1) mv[hole++].y = s0 + __ffsll(holes) - 1;
      for (; movers; movers &= movers - 1) mv[mover++].x = s0 + __ffsll(movers) - 1;
    }
  }
  if (tid == 0) a.count[u] = moved;
  __syncthreads();
  int2* list = KEYS ? reinterpret_cast<int2*>(s_key) : mv;  // a move takes one of two slots: it fits
  for (int j = tid; j < moved; j += NT) {
    const int2 m = mv[j];
    if (KEYS) list[j] = m;
    wo[m.y] = w[m.x];
    po[m.y] = p[m.x];
  }
  __syncthreads();
  if (!copy_w || !copy_p) {                // the survivors have been read
    for (int i = fin + tid; i < a.S; i += NT) {
      if (!copy_w) wo[i] = 0.f;
      if (!copy_p) po[i] = -1;
    }
  }
  if (!moves_here) return;
  if (a.lengths_out != a.lengths && u < (long)a.B * a.nkv && h == 0 && tid == 0) a.lengths_out[b] = fin;
  // short units want more blocks on an SM (32 registers), long ones more rows in flight
  move_rows<NT == 256 ? 1 : 2>(a, list, u, moved, tid, NT);
}

// the rows of all units, `parts` blocks each, and the new lengths; parts 0: the lengths only
__global__ void __launch_bounds__(256) evict_move_k(KvEvictArgs a, int parts) {
  join_wait();
  if (blockIdx.x == 0)
    for (int b = threadIdx.x; b < a.B; b += 256) a.lengths_out[b] = min(min(max(a.lengths[b], 0), a.S), a.keep);
  if (parts == 0) return;
  const long u = blockIdx.x / parts;
  move_rows<2>(a, a.moves + u * a.keep, u, a.count[u], (int)(blockIdx.x % parts) * 256 + threadIdx.x, 256 * parts);
}

constexpr int CT = 256, CMAX = 1024;

template <typename V>
__global__ void __launch_bounds__(CT) commit_k(KvCommitArgs a) {
  __shared__ int s_par[CMAX], s_path[CMAX];
  __shared__ long s_tok[CMAX], s_tgt[CMAX];
  __shared__ int s_cnt;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = blockIdx.x % a.B, n = blockIdx.x / a.B;
  const int len = min(max(a.lengths[b], 0), a.S), fit = min(a.T, a.S - len);   // nodes whose rows are in the cache
  for (int i = tid; i < a.T; i += CT) {
    s_par[i] = a.parents[b * a.par_b + i];
    s_tok[i] = a.tokens[(long)b * a.T + i];
    s_tgt[i] = a.targets[(long)b * a.T + i];
  }
  __syncthreads();
  if (warp == 0) {
    int cur = 0, cnt = fit > 0;
    if (lane == 0) s_path[0] = 0;
    while (true) {
      const long want = s_tgt[cur];
      int found = -1;
      for (int i0 = (cur + 1) & ~31; i0 < fit && found < 0; i0 += 32) {   // nodes above cur only: the walk ends
        const int i = i0 + lane;
        const bool on = i > cur && i < fit && s_par[i] == cur && s_tok[i] == want;
        const unsigned any = __ballot_sync(0xffffffffu, on);
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
        a.next[b] = cnt ? s_tgt[cur] : s_tok[0];
      }
    }
  }
  __syncthreads();
  const int cnt = s_cnt;
  if (n == 0)
    for (int i = tid; i < a.T; i += CT) a.path[(long)b * a.T + i] = i < cnt ? s_path[i] : -1;

  // rows: a thread owns one column block of one head's K or V rows and moves them in order, eight loads
  // at a time (a destination never lies behind a later source)
  const int C = a.hd * a.esize / (int)sizeof(V);
  for (int i = tid; i < 2 * a.nkv * C; i += CT) {
    if (i >= a.nkv * C && a.vc == a.kc) break;           // one tensor for keys and values moves once
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
        if (j0 + j < cnt) x[j] = *reinterpret_cast<const V*>(base + s_path[j0 + j] * rs);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j0 + j < cnt) *reinterpret_cast<V*>(base + (j0 + j) * rs) = x[j];
    }
  }
  for (int h = warp; h < a.nkv; h += CT / 32) {
    float* wt = a.weight ? a.weight + n * a.w_n + b * a.w_b + h * a.w_h + len : nullptr;
    int* ps = a.positions ? a.positions + n * a.p_n + b * a.p_b + h * a.p_h + len : nullptr;
    for (int j0 = 0; j0 < fit; j0 += 32) {
      const int j = j0 + lane;
      const bool on = j < cnt;
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

template <int NT, bool KEYS>
static int select_units(const KvEvictArgs& a, unsigned units, int moves_here, cudaStream_t st) {
  const size_t sm = KEYS ? (size_t)a.S * 4 + 8 : 0;
  const cudaError_t e = cudaFuncSetAttribute(s0::kv::evict_k<NT, KEYS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sm);
  if (e != cudaSuccess) return (int)e;
  s0::kv::evict_k<NT, KEYS><<<units, NT, sm, st>>>(a, moves_here);
  return s0::kv::launched();
}

int kv_evict_launch(KvEvictArgs a, cudaStream_t st) {
  using namespace s0::kv;
  const long units = (long)a.N * a.B * a.nkv;
  if (units <= 0) return 0;
  a.width = width_of(a.hd, a.esize, {a.kc_n, a.kc_b, a.kc_h, a.kc_s, a.vc_n, a.vc_b, a.vc_h, a.vc_s}, {a.kc, a.vc});
  const bool here = units >= a.sms;                        // enough units to keep the memory busy by themselves
  // Threads per unit: keys of more than 24 KB leave no more than six blocks on an SM whatever their size, so
  // those are larger; few units on an otherwise empty GPU take still more.  200 KB of keys at most.
  const bool fits = a.S <= 50 * 1024;
  const unsigned n = (unsigned)units;
  const int rc = !fits ? select_units<512, false>(a, n, here, st)
                 : a.S <= 6 * 1024 && (here || a.S <= 2048) ? select_units<256, true>(a, n, here, st)
                 : here ? select_units<512, true>(a, n, here, st) : select_units<1024, true>(a, n, here, st);
  if (rc || (here && a.lengths_out != a.lengths)) return rc;
  // lengths that are overwritten in place wait for all units to have read them
  const int parts = here ? 0 : (int)std::max<long>(1, std::min<long>(32, (8L * a.sms + units - 1) / units));
  return launch_after(evict_move_k, parts ? (unsigned)(units * parts) : 1u, 256, st, a, parts);
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
  return launched();
}
