// Attention of a few new tokens over a 16-bit key / value cache on the tensor cores (the operator is
// described in kv_attention.cu; heads up to 128 wide, 16-byte aligned rows).
//
// What bounds it: a step reads every cached key and value once and does 4 T group flops per element
// pair, so up to some 64 rows (new tokens x query heads of a key head) it is bound by HBM.  Both kernels
// therefore keep a ring of key / value tiles in flight by cp.async all the time, across the ends of
// units: a CTA's tiles (see kv_attention.cuh) form one stream, and the loads run ahead of the
// products without regard to which unit a tile belongs to.
//   kv_attn_few_k    up to 16 rows: every warp streams key slabs of its own (16 keys of 128, 32 of 64
//                    channels) through its own ring, with a running maximum and sum of its own and no
//                    barrier; the four warps' results are joined at the end of a unit;
//   kv_attn_rows_k   more rows: the warps of a CTA take 16 rows each and share the tiles.
// Products: mma.m16n8k16 with fp32 accumulators.  The scores never leave registers; p is rounded to the
// cache's type for the second product (relative error u, as the output's own rounding), while the sum
// of the row is taken from the unrounded values in fp32.
#include <algorithm>

#include "kv_attention.cuh"

namespace s0 {
namespace kv {

template <typename T> S0_DEV uint32_t pack2(float lo, float hi);
template <> S0_DEV uint32_t pack2<__nv_bfloat16>(float lo, float hi) { return pack_bf16(lo, hi); }
template <> S0_DEV uint32_t pack2<__half>(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <typename T> S0_DEV void mma16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1);
template <> S0_DEV void mma16<__nv_bfloat16>(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) { mma_bf16(c, a, b0, b1); }
template <> S0_DEV void mma16<__half>(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// exponent bits all ones: infinity or NaN
template <typename T> struct Inf;
template <> struct Inf<__nv_bfloat16> { static constexpr uint32_t mask = 0x7f80u; };
template <> struct Inf<__half> { static constexpr uint32_t mask = 0x7c00u; };
template <typename T> S0_DEV bool any_inf(uint4 x) {
  constexpr uint32_t m = Inf<T>::mask, hi = m << 16;
  auto bad = [](uint32_t v) { return (v & m) == m || (v & hi) == hi; };
  return bad(x.x) || bad(x.y) || bad(x.z) || bad(x.w);
}

// byte offset of 16-byte chunk c of row r in a tile of HD 16-bit channels: the chunks of eight
// consecutive rows fall into eight different groups of banks
template <int HD> S0_DEV int tile_at(int r, int c) { return r * HD * 2 + ((c ^ (r & 7)) << 4); }

// B fragments of two 8-key groups (rows n0 .. n0 + 15) at channels k0 .. k0 + 15 of a K tile
template <int HD> S0_DEV void frag_k(uint32_t* f, const char* tile, int n0, int k0, int lane) {
  const int j = lane >> 3, r = n0 + (lane & 7) + (j >> 1) * 8, c = (k0 >> 3) + (j & 1);
  ldsm_x4(f[0], f[1], f[2], f[3], tile + tile_at<HD>(r, c));
}
// B fragments of two 8-channel groups (n0 .. n0 + 15) at keys k0 .. k0 + 15 of a V tile
template <int HD> S0_DEV void frag_v(uint32_t* f, const char* tile, int n0, int k0, int lane) {
  const int j = lane >> 3, r = k0 + (lane & 7) + (j & 1) * 8, c = (n0 >> 3) + (j >> 1);
  ldsm_x4_t(f[0], f[1], f[2], f[3], tile + tile_at<HD>(r, c));
}

// A unit and the place in it; steps from unit to unit in the plan's order.
struct Cur {
  int b, u, len, n, t;  // sequence, head * nrb + row block, cached tokens, tiles, tile
};
S0_DEV void cur_set(Cur& c, const KvAttnArgs& a, int KT) {
  c.len = cached(a, c.b);
  c.n = tiles_of(a, c.len, KT);
}
S0_DEV void cur_next_unit(Cur& c, const KvAttnArgs& a, int KT) {
  if (++c.u == a.nkv * a.nrb) {
    c.u = 0;
    if (++c.b < a.B) cur_set(c, a, KT);
  }
}
S0_DEV void cur_skip(Cur& c, const KvAttnArgs& a, int KT, int by) {
  c.t += by;
  while (c.b < a.B && c.t >= c.n) {
    c.t -= c.n;
    cur_next_unit(c, a, KT);
  }
}

// The first tile of this CTA and how many it has.  a.whole: one unit per CTA (caches that are short
// enough); otherwise the even split.  Leaves the prefix table behind in `scratch` (B + 33 ints).
S0_DEV long cta_share(Cur& c, const KvAttnArgs& a, int KT, int* scratch, int ctas) {
  const int hr = a.nkv * a.nrb;
  if (a.whole) {
    c.b = blockIdx.x / hr;
    c.u = blockIdx.x - c.b * hr;
    c.t = 0;
    cur_set(c, a, KT);
    return c.n;
  }
  const Plan p = make_plan(a, plan_prefix(a, KT, scratch), ctas, a.min_per);
  const long w = (long)blockIdx.x * p.per;
  if (w >= p.total) return 0;
  const Seg s = find_seg(a, scratch, w, KT);
  c.b = s.b;
  c.u = s.h * a.nrb + s.rb;
  c.len = s.len;
  c.n = s.n;
  c.t = s.t0;
  return min(p.total - w, p.per);
}

// where row `row` of the unit lies in q / o: element offset of its first channel
S0_DEV long out_at(const KvAttnArgs& a, int b, int h, int row) {
  const int t = row / a.group, g = row - t * a.group;
  return (((long)b * a.T + t) * a.nkv * a.group + h * a.group + g) * a.hd;
}
template <typename T> S0_DEV const T* q_at(const KvAttnArgs& a, int b, int h, int row) {
  const int t = row / a.group, g = row - t * a.group;
  return (const T*)a.q + b * a.q_b + t * a.q_t + (long)(h * a.group + g) * a.q_h;
}

// A fragments of rows [r0, r0 + 16) straight from global memory; rows past R and channels past hd are 0
template <typename T, int HD>
S0_DEV void load_q(uint32_t (*qf)[4], const KvAttnArgs& a, int b, int h, int r0, int R, int lane) {
  const int g = lane >> 2, t = lane & 3;
  const T* p0 = r0 + g < R ? q_at<T>(a, b, h, r0 + g) : nullptr;
  const T* p1 = r0 + g + 8 < R ? q_at<T>(a, b, h, r0 + g + 8) : nullptr;
#pragma unroll
  for (int k = 0; k < HD / 16; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const T* p = e & 1 ? p1 : p0;
      const int d = k * 16 + (e >> 1) * 8 + 2 * t;
      qf[k][e] = p && d < a.hd ? *reinterpret_cast<const uint32_t*>(p + d) : 0u;
    }
}

// A tile of new tokens: hidden rows' NaNs and infinities must not meet their zero probabilities in the
// product, so what is not finite in V is added by hand to the rows that see it, and taken out of the
// tile.  `own(e)`: this thread's rows; NK keys.  Rare: only tiles that hold such a value come here.
template <typename T, int HD, int NK>
S0_DEV void add_infinities(float (*o)[4], char* tv, const KvAttnArgs& a, int b, int row0, int R, int k0, int nk, int lane) {
  const int g = lane >> 2, t = lane & 3;
  for (int j = 0; j < nk; ++j)
#pragma unroll
    for (int nt = 0; nt < HD / 8; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = row0 + g + (e >> 1) * 8, d = nt * 8 + 2 * t + (e & 1);
        const unsigned short x = *reinterpret_cast<const unsigned short*>(tv + tile_at<HD>(j, nt) + (2 * t + (e & 1)) * 2);
        if ((x & Inf<T>::mask) == Inf<T>::mask && row < R && d < a.hd && sees(a, b, row / a.group, k0 + j))
          o[nt][e] += Elem<T>::to(*reinterpret_cast<const T*>(&x));
      }
}
template <typename T, int HD, int NK>
S0_DEV void drop_infinities(char* tv, int i0, int step) {
  for (int i = i0; i < NK * HD; i += step) {
    const int j = i / HD, d = i - j * HD;
    unsigned short* p = reinterpret_cast<unsigned short*>(tv + tile_at<HD>(j, d >> 3) + (d & 7) * 2);
    if ((*p & Inf<T>::mask) == Inf<T>::mask) *p = 0;
  }
}

// Softmax of a warp's 16 x NK scores in place, with the running statistics and the rescaled output.
// Rows g and g + 8 of the block at row0; keys k0 + ... of which nk exist.
template <typename T, int HD, int NK>
S0_DEV void softmax_tile(float (*s)[4], float (*o)[4], float* m, float* l, const KvAttnArgs& a, int b, long bh, int row0,
                         int R, bool tail, int len, int k0, int nk, int lane) {
  const int g = lane >> 2, t = lane & 3;
  const bool part = tail || nk < NK;
#pragma unroll
  for (int nt = 0; nt < NK / 8; ++nt)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float x = s[nt][e] * a.scale_log2;
      if (part) {
        const int j = nt * 8 + 2 * t + (e & 1), row = row0 + g + (e >> 1) * 8;
        if (j >= nk || (tail && (row >= R || !sees(a, b, row / a.group, k0 + j)))) x = -CUDART_INF_F;
      }
      s[nt][e] = x;
    }
  if (a.scores) {
#pragma unroll
    for (int nt = 0; nt < NK / 8; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int j = nt * 8 + 2 * t + (e & 1), row = row0 + g + (e >> 1) * 8;
        if (j < nk && row < R) a.scores[(bh * R + row) * a.sp + (tail ? len : 0) + k0 + j] = s[nt][e];
      }
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    float mx = m[r];
#pragma unroll
    for (int nt = 0; nt < NK / 8; ++nt) mx = fmaxf(mx, fmaxf(s[nt][2 * r], s[nt][2 * r + 1]));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    const float base = mx == -CUDART_INF_F ? 0.f : mx;   // a row that has seen nothing yet
    const float al = exp2f(m[r] - base);
    m[r] = mx;
    float sum = 0.f;
#pragma unroll
    for (int nt = 0; nt < NK / 8; ++nt) {
      s[nt][2 * r] = exp2f(s[nt][2 * r] - base);
      s[nt][2 * r + 1] = exp2f(s[nt][2 * r + 1] - base);
      sum += s[nt][2 * r] + s[nt][2 * r + 1];
    }
    l[r] = l[r] * al + sum;                              // this lane's share; joined at the end
#pragma unroll
    for (int i = 0; i < HD / 8; ++i) {
      o[i][2 * r] *= al;
      o[i][2 * r + 1] *= al;
    }
  }
}

// a finished unit's or a piece's rows from the accumulators
template <typename T, int HD>
S0_DEV void write_rows(float (*o)[4], const float* m, const float* l, const KvAttnArgs& a, int b, int h, int r0, int row0, int R,
                       bool all, long slot, int lane) {
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int row = row0 + g + 8 * r;
    if (row >= R) continue;
    if (all) {
      const float inv = l[r] == 0.f ? 0.f : 1.f / l[r];
      T* p = (T*)a.o + out_at(a, b, h, row);
#pragma unroll
      for (int nt = 0; nt < HD / 8; ++nt)
        if (nt * 8 < a.hd)
          *reinterpret_cast<uint32_t*>(p + nt * 8 + 2 * t) = pack2<T>(o[nt][2 * r] * inv, o[nt][2 * r + 1] * inv);
      if (a.lse && t == 0) a.lse[((long)b * a.nkv + h) * R + row] = lse2(m[r], l[r]);
    } else {
      const long at = slot * a.rows + row - r0;
#pragma unroll
      for (int nt = 0; nt < HD / 8; ++nt)
        if (nt * 8 < a.hd)
          *reinterpret_cast<float2*>(a.part_o + at * a.hd + nt * 8 + 2 * t) = make_float2(o[nt][2 * r], o[nt][2 * r + 1]);
      if (t == 0) *reinterpret_cast<float2*>(a.part_ml + at * 2) = make_float2(m[r], l[r]);
    }
  }
}

// One tile of a unit's stream into a stage: K rows, then V rows; what does not exist becomes 0.
template <typename T, int HD, int NK, int NT>
S0_DEV void load_tile(char* st, const KvAttnArgs& a, const Cur& c, int tid) {
  constexpr int C = HD / 8, RS = NT / C;               // chunks of a row, rows per pass
  const int ncache = (c.len + NK - 1) / NK, h = c.u / a.nrb;
  const bool tail = c.t >= ncache;
  const int k0 = (tail ? c.t - ncache : c.t) * NK, nk = (tail ? a.T : c.len) - k0;
  const int ch = tid % C, r0 = tid / C;
  const long ks = tail ? a.kn_t : a.kc_s, vs = tail ? a.vn_t : a.vc_s;
  const T* k = tail ? (const T*)a.kn + c.b * a.kn_b + h * a.kn_h : (const T*)a.kc + c.b * a.kc_b + h * a.kc_h;
  const T* v = tail ? (const T*)a.vn + c.b * a.vn_b + h * a.vn_h : (const T*)a.vc + c.b * a.vc_b + h * a.vc_h;
  const bool in = ch * 8 < a.hd;
  k += (in ? ch * 8 : 0) + (k0 + r0) * ks;
  v += (in ? ch * 8 : 0) + (k0 + r0) * vs;
#pragma unroll
  for (int i = 0; i < NK / RS; ++i) {
    const int r = r0 + i * RS;
    const bool ok = in && r < nk;
    cp_async16(st + tile_at<HD>(r, ch), ok ? k + (long)i * RS * ks : a.q, ok ? 16 : 0);
    cp_async16(st + NK * HD * 2 + tile_at<HD>(r, ch), ok ? v + (long)i * RS * vs : a.q, ok ? 16 : 0);
  }
}

// stores a tile of new rows behind the cached ones
template <typename T, int HD, int NK>
S0_DEV void put_tile(const char* st, const KvAttnArgs& a, int b, int h, int len, int k0, int nk, int i0, int step) {
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

constexpr int FW = 4, FS = 3;  // warps of a block, stages of a warp's ring

template <int HD> constexpr int few_keys() { return HD == 128 ? 16 : 32; }
template <int HD> constexpr int few_stage() { return 2 * few_keys<HD>() * HD * 2; }

template <typename T, int HD>
__global__ void __launch_bounds__(32 * FW, 2) kv_attn_few_k(KvAttnArgs a, int ctas) {
  constexpr int NK = few_keys<HD>(), SB = few_stage<HD>(), OLD = HD + 4;
  extern __shared__ __align__(128) char smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int R = a.T * a.group, mrows = min(16, R);
  char* ring = smem + warp * FS * SB;
  float* sO = reinterpret_cast<float*>(smem + FW * FS * SB);   // [2][mrows][OLD] outputs of two warps
  float* sM = sO + 2 * mrows * OLD;                            // [2][mrows][2] maxima, sums
  Cur cur;
  const long share = cta_share(cur, a, NK, reinterpret_cast<int*>(smem), ctas);
  __syncthreads();                                             // the plan's scratch becomes the ring
  if (share <= 0) return;

  Cur ahead = cur;                                             // this warp's next tile to load
  long left = (share - warp + FW - 1) / FW;
  cur_skip(ahead, a, NK, warp);
  auto fetch = [&](int stage) {
    if (left > 0) {
      load_tile<T, HD, NK, 32>(ring + stage * SB, a, ahead, lane);
      if (--left > 0) cur_skip(ahead, a, NK, FW);
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < FS - 1; ++i) fetch(i);

  long done = 0;                                               // tiles of the share before this unit
  int stage = 0;
  long mine = warp;                                            // this warp's next tile of the share
  while (done < share) {
    const int b = cur.b, h = cur.u / a.nrb, rb = cur.u - h * a.nrb, r0 = rb * 16;
    const long bh = (long)b * a.nkv + h;
    const int t1 = (int)min((long)cur.n, cur.t + (share - done));
    const int ncache = (cur.len + NK - 1) / NK;
    const long end = done + (t1 - cur.t);
    uint32_t qf[HD / 16][4];
    load_q<T, HD>(qf, a, b, h, r0, R, lane);
    float o[HD / 8][4];
#pragma unroll
    for (int i = 0; i < HD / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m[2] = {-CUDART_INF_F, -CUDART_INF_F}, l[2] = {0.f, 0.f};

    for (; mine < end; mine += FW) {
      const int tt = cur.t + (int)(mine - done);
      __syncwarp();                                            // the stage that is loaded next has been read
      fetch(stage == 0 ? FS - 1 : stage - 1);
      cp_async_wait_group<FS - 1>();
      __syncwarp();
      char* st = ring + stage * SB;
      const bool tail = tt >= ncache;
      const int k0 = (tail ? tt - ncache : tt) * NK, nk = min(NK, (tail ? a.T : cur.len) - k0);
      float s[NK / 8][4];
#pragma unroll
      for (int i = 0; i < NK / 8; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
#pragma unroll
      for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
        for (int np = 0; np < NK / 16; ++np) {
          uint32_t f[4];
          frag_k<HD>(f, st, np * 16, kk * 16, lane);
          mma16<T>(s[2 * np], qf[kk], f[0], f[1]);
          mma16<T>(s[2 * np + 1], qf[kk], f[2], f[3]);
        }
      softmax_tile<T, HD, NK>(s, o, m, l, a, b, bh, r0, R, tail, cur.len, k0, nk, lane);
      char* tv = st + NK * HD * 2;
      if (tail) {
        if (rb == 0) put_tile<T, HD, NK>(st, a, b, h, cur.len, k0, nk, lane, 32);
        bool bad = false;
        for (int i = lane; i < NK * HD / 8; i += 32) bad |= any_inf<T>(*reinterpret_cast<const uint4*>(tv + i * 16));
        if (__any_sync(0xffffffffu, bad)) {
          add_infinities<T, HD, NK>(o, tv, a, b, r0, R, k0, nk, lane);
          __syncwarp();
          drop_infinities<T, HD, NK>(tv, lane, 32);
          __syncwarp();
        }
      }
#pragma unroll
      for (int kk = 0; kk < NK / 16; ++kk) {
        uint32_t pa[4];
        pa[0] = pack2<T>(s[2 * kk][0], s[2 * kk][1]);
        pa[1] = pack2<T>(s[2 * kk][2], s[2 * kk][3]);
        pa[2] = pack2<T>(s[2 * kk + 1][0], s[2 * kk + 1][1]);
        pa[3] = pack2<T>(s[2 * kk + 1][2], s[2 * kk + 1][3]);
#pragma unroll
        for (int dp = 0; dp < HD / 16; ++dp) {
          uint32_t f[4];
          frag_v<HD>(f, tv, dp * 16, kk * 16, lane);
          mma16<T>(o[2 * dp], pa, f[0], f[1]);
          mma16<T>(o[2 * dp + 1], pa, f[2], f[3]);
        }
      }
      stage = stage == FS - 1 ? 0 : stage + 1;
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    }
    // join the warps: 2 and 3 hand over to 0 and 1, then 1 to 0
    auto give = [&](int slot) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int row = g + 8 * r;
        if (row >= mrows) continue;
        float* p = sO + (slot * mrows + row) * OLD + 2 * t;
#pragma unroll
        for (int nt = 0; nt < HD / 8; ++nt) *reinterpret_cast<float2*>(p + nt * 8) = make_float2(o[nt][2 * r], o[nt][2 * r + 1]);
        if (t == 0) {
          sM[(slot * mrows + row) * 2] = m[r];
          sM[(slot * mrows + row) * 2 + 1] = l[r];
        }
      }
    };
    auto take = [&](int slot) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int row = g + 8 * r;
        if (row >= mrows) continue;
        const float m2 = sM[(slot * mrows + row) * 2], l2 = sM[(slot * mrows + row) * 2 + 1];
        const float mx = fmaxf(m[r], m2), base = mx == -CUDART_INF_F ? 0.f : mx;
        const float e0 = exp2f(m[r] - base), e1 = exp2f(m2 - base);
        m[r] = mx;
        l[r] = l[r] * e0 + l2 * e1;
        const float* p = sO + (slot * mrows + row) * OLD + 2 * t;
#pragma unroll
        for (int nt = 0; nt < HD / 8; ++nt) {
          const float2 x = *reinterpret_cast<const float2*>(p + nt * 8);
          o[nt][2 * r] = o[nt][2 * r] * e0 + x.x * e1;
          o[nt][2 * r + 1] = o[nt][2 * r + 1] * e0 + x.y * e1;
        }
      }
    };
    if (warp >= 2) give(warp - 2);
    __syncthreads();
    if (warp < 2) take(warp);
    if (warp == 1) {
      __syncwarp();
      give(1);                                                 // slot 1 is read by this warp only
    }
    __syncthreads();
    if (warp == 0) {
      take(1);
      const bool first = cur.t == 0, all = first && t1 == cur.n;
      write_rows<T, HD>(o, m, l, a, b, h, r0, r0, R, all, 2L * blockIdx.x + (first ? 1 : 0), lane);
    }
    done = end;
    cur.t = 0;
    cur_next_unit(cur, a, NK);
  }
}

// WR warps of 16 rows each
template <int HD> constexpr int rows_keys() { return 64; }

template <typename T, int HD, int WR, int ST>
__global__ void __launch_bounds__(32 * WR, WR == 8 ? 1 : 2) kv_attn_rows_k(KvAttnArgs a, int ctas) {
  constexpr int NK = rows_keys<HD>(), SB = 2 * NK * HD * 2, NT = 32 * WR;
  extern __shared__ __align__(128) char smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int R = a.T * a.group;
  Cur cur;
  const long share = cta_share(cur, a, NK, reinterpret_cast<int*>(smem), ctas);
  __syncthreads();
  if (share <= 0) return;
  Cur ahead = cur;
  long left = share;
  auto fetch = [&](int stage) {
    if (left > 0) {
      load_tile<T, HD, NK, NT>(smem + stage * SB, a, ahead, tid);
      if (--left > 0) cur_skip(ahead, a, NK, 1);
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < ST - 1; ++i) fetch(i);

  long done = 0;
  int stage = 0;
  while (done < share) {
    const int b = cur.b, h = cur.u / a.nrb, rb = cur.u - h * a.nrb, r0 = rb * 16 * WR, row0 = r0 + 16 * warp;
    const long bh = (long)b * a.nkv + h;
    const int t1 = (int)min((long)cur.n, cur.t + (share - done));
    const int ncache = (cur.len + NK - 1) / NK;
    uint32_t qf[HD / 16][4];
    load_q<T, HD>(qf, a, b, h, row0, R, lane);
    float o[HD / 8][4];
#pragma unroll
    for (int i = 0; i < HD / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m[2] = {-CUDART_INF_F, -CUDART_INF_F}, l[2] = {0.f, 0.f};
    for (int tt = cur.t; tt < t1; ++tt) {
      cp_async_wait_group<ST - 2>();
      __syncthreads();                                         // the tile is there, and the one before it has been read
      fetch(stage == 0 ? ST - 1 : stage - 1);
      char* st = smem + stage * SB;
      char* tv = st + NK * HD * 2;
      const bool tail = tt >= ncache;
      const int k0 = (tail ? tt - ncache : tt) * NK, nk = min(NK, (tail ? a.T : cur.len) - k0);
      float s[NK / 8][4];
#pragma unroll
      for (int i = 0; i < NK / 8; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
#pragma unroll
      for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
        for (int np = 0; np < NK / 16; ++np) {
          uint32_t f[4];
          frag_k<HD>(f, st, np * 16, kk * 16, lane);
          mma16<T>(s[2 * np], qf[kk], f[0], f[1]);
          mma16<T>(s[2 * np + 1], qf[kk], f[2], f[3]);
        }
      softmax_tile<T, HD, NK>(s, o, m, l, a, b, bh, row0, R, tail, cur.len, k0, nk, lane);
      if (tail) {
        if (rb == 0) put_tile<T, HD, NK>(st, a, b, h, cur.len, k0, nk, tid, NT);
        bool bad = false;
        for (int i = tid; i < NK * HD / 8; i += NT) bad |= any_inf<T>(*reinterpret_cast<const uint4*>(tv + i * 16));
        if (__syncthreads_or(bad)) {
          add_infinities<T, HD, NK>(o, tv, a, b, row0, R, k0, nk, lane);
          __syncthreads();
          drop_infinities<T, HD, NK>(tv, tid, NT);
          __syncthreads();
        }
      }
#pragma unroll
      for (int kk = 0; kk < NK / 16; ++kk) {
        uint32_t pa[4];
        pa[0] = pack2<T>(s[2 * kk][0], s[2 * kk][1]);
        pa[1] = pack2<T>(s[2 * kk][2], s[2 * kk][3]);
        pa[2] = pack2<T>(s[2 * kk + 1][0], s[2 * kk + 1][1]);
        pa[3] = pack2<T>(s[2 * kk + 1][2], s[2 * kk + 1][3]);
#pragma unroll
        for (int dp = 0; dp < HD / 16; ++dp) {
          uint32_t f[4];
          frag_v<HD>(f, tv, dp * 16, kk * 16, lane);
          mma16<T>(o[2 * dp], pa, f[0], f[1]);
          mma16<T>(o[2 * dp + 1], pa, f[2], f[3]);
        }
      }
      stage = stage == ST - 1 ? 0 : stage + 1;
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    }
    const bool first = cur.t == 0, all = first && t1 == cur.n;
    write_rows<T, HD>(o, m, l, a, b, h, r0, row0, R, all, 2L * blockIdx.x + (first ? 1 : 0), lane);
    done += t1 - cur.t;
    cur.t = 0;
    cur_next_unit(cur, a, NK);
  }
}

template <typename K>
int run_k(K k, const KvAttnArgs& a, int threads, size_t sm, cudaStream_t st) {
  const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sm);
  if (e != cudaSuccess) return (int)e;
  const int grid = a.whole ? a.B * a.nkv * a.nrb : a.ctas;
  k<<<grid, threads, sm, st>>>(a, a.ctas);
  return (int)cudaGetLastError();
}

template <typename T, int HD>
int launch_tc(const KvAttnArgs& a, cudaStream_t st) {
  const size_t plan = (size_t)(a.B + 33) * 4;
  if (a.rows == 16) {
    const int mrows = std::min(16, a.T * a.group);
    const size_t sm = FW * FS * few_stage<HD>() + (size_t)2 * mrows * (HD + 4 + 2) * 4;
    return run_k(kv_attn_few_k<T, HD>, a, 32 * FW, std::max(sm, plan), st);
  }
  constexpr int SB = 2 * rows_keys<HD>() * HD * 2;
  if (a.rows == 32) return run_k(kv_attn_rows_k<T, HD, 2, 3>, a, 64, std::max<size_t>(3 * SB, plan), st);
  if (a.rows == 64) return run_k(kv_attn_rows_k<T, HD, 4, 3>, a, 128, std::max<size_t>(3 * SB, plan), st);
  return run_k(kv_attn_rows_k<T, HD, 8, 4>, a, 256, std::max<size_t>(4 * SB, plan), st);
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
  const int R = a.T * a.group, few = a.hd > 64 ? s0::kv::few_keys<128>() : s0::kv::few_keys<64>();
  a.rows = R <= 16 ? 16 : R <= 32 ? 32 : R <= 64 ? 64 : 128;
  a.nrb = (R + a.rows - 1) / a.rows;
  a.tile = a.rows == 16 ? few : 64;
  a.ctas = (a.rows == 128 ? 1 : 2) * sms;
  a.min_per = a.rows == 16 ? 4 : 1;
  a.whole = 0;
}

int kv_attn_tc_launch(const KvAttnArgs& a, int dtype, cudaStream_t st) {
  using namespace s0::kv;
  if (dtype == 1) return a.hd > 64 ? launch_tc<__half, 128>(a, st) : launch_tc<__half, 64>(a, st);
  return a.hd > 64 ? launch_tc<__nv_bfloat16, 128>(a, st) : launch_tc<__nv_bfloat16, 64>(a, st);
}
