// Masked, capped and biased 16-bit attention and its shared-prefix form: entry points,
// work split, the id ranges of key tiles and the merge of split rows.  The attention kernel
// is in masked_attn.cuh.
#include "masked_attn.cuh"

#include <algorithm>
#include <cfloat>

namespace qf2 {
namespace mattn {

// Set by a kernel whose bounded wait gave up; read and cleared by qf2_masked_attn_status.
// It lives in the module, zero when loaded, so that a call needs no launch to clear one.
__device__ int g_status;

// Failure-injection settings of the launches (qf2_masked_attn_fault_injection).
static std::atomic<long long> g_wait_clocks{kWaitClocks};
static std::atomic<int> g_skip_kv{-1};

// ------------------------------------------------------------- key ids --
// What the attention kernel wants to know of ids, in one launch.  grid (kb + qb, B), 1024 threads.
// The first kb blocks of a batch element: a padded copy of the key ids (tiles of 128, pad -2; of
// 64-bit ids the low words, then the high ones, a negative id as -1) and the least and greatest
// entry of each tile, eight tiles a block.
// The other qb blocks, 1024 queries each: whether the key ids never fall (as unsigned numbers, so
// that the negative ids of padding come last), which each block sees for itself; then the keys of
// a query's id are one run, found here, and the attention kernel masks by ranges and looks at no
// id.  A warp takes 32 queries, one id among them at a time: the tiles whose first key comes
// before the id are counted, then such keys of the last of these tiles.
template <typename I>
__global__ void __launch_bounds__(1024) mattn_ids_kernel(const I* __restrict__ q_ids, const I* __restrict__ k_ids,
                                                         int Sq, int Skv, int nto, int kb, int32_t* __restrict__ copy,
                                                         int64_t hi_off, int2* __restrict__ k_rng,
                                                         int2* __restrict__ q_rng, int* __restrict__ order) {
  using U = std::make_unsigned_t<I>;
  grid_launch_dependents();
  const int b = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const I* k = k_ids + (int64_t)b * Skv;
  if ((int)blockIdx.x < kb) {
    const int j = blockIdx.x * 1024 + threadIdx.x, t = j / kBlk;
    const I id = j < Skv ? k[j] : -2;
    const int v = sizeof(I) == 8 && j < Skv && id < 0 ? -1 : (int)id;
    __shared__ int2 part[32];
    const int mn = __reduce_min_sync(0xffffffffu, v), mx = __reduce_max_sync(0xffffffffu, v);
    if (lane == 0) part[warp] = make_int2(mn, mx);
    __syncthreads();
    if (t >= nto) return;
    copy[(int64_t)b * nto * kBlk + j] = v;
    if constexpr (sizeof(I) == 8) copy[hi_off + (int64_t)b * nto * kBlk + j] = (int)(id >> 32);
    if ((threadIdx.x & (kBlk - 1)) == 0) {
      const int2 p0 = part[warp], p1 = part[warp + 1], p2 = part[warp + 2], p3 = part[warp + 3];
      k_rng[(int64_t)b * nto + t] = make_int2(min(min(p0.x, p1.x), min(p2.x, p3.x)), max(max(p0.y, p1.y), max(p2.y, p3.y)));
    }
    return;
  }
  const int i = (blockIdx.x - kb) * 1024 + threadIdx.x;
  const I id = i < Sq ? q_ids[(int64_t)b * Sq + i] : -1;
  int fine = 1, wide = 0;
#pragma unroll 4
  for (int j = threadIdx.x; j < Skv - 1; j += 1024) {
    fine &= (U)k[j] <= (U)k[j + 1];
    if constexpr (sizeof(I) == 8) wide |= k[j] > 0x7fffffff;
  }
  fine = __syncthreads_and(fine);
  if (sizeof(I) == 8 && !fine) wide = __syncthreads_or(wide || k[Skv - 1] > 0x7fffffff);
  // (out of order and all below 2^31, 64-bit ids are compared by their low words alone)
  if ((int)blockIdx.x == kb && threadIdx.x == 0) order[b] = fine ? kInOrder : wide ? kMixedWide : kMixed;
  if (!fine) return;
  // keys of less than x (as unsigned numbers), by the warp
  auto below = [&](U x) -> int {
    int tiles = 0;
    for (int t = lane; t < nto; t += 32) tiles += (U)k[(int64_t)t * kBlk] < x;
    tiles = __reduce_add_sync(0xffffffffu, tiles);
    if (tiles == 0) return 0;
    int n = 0;
#pragma unroll
    for (int u = 0; u < kBlk; u += 32) {
      const int j = (tiles - 1) * kBlk + u + lane;
      n += j < Skv && (U)k[j] < x;
    }
    return (tiles - 1) * kBlk + __reduce_add_sync(0xffffffffu, n);
  };
  int2 r = make_int2(0, 0);
  uint32_t left = __ballot_sync(0xffffffffu, id >= 0);
  while (left) {
    const I x = __shfl_sync(0xffffffffu, id, __ffs(left) - 1);
    const int lo = below((U)x), hi = below((U)x + 1u);
    if (id == x) r = make_int2(lo, hi);
    left &= ~__ballot_sync(0xffffffffu, id == x);
  }
  if (i < Sq) q_rng[(int64_t)b * Sq + i] = r;
}

// ----------------------------------------------------------- merge splits --
// out = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s over the splits of one row (a split
// that saw nothing has m = -inf and is not read).  One CTA per (batch, token, head) row:
// D / 4 threads cover the row in 16-byte pieces, 128 / (D / 4) such groups take every
// second, fifth, ... split, and the groups are added in a fixed order.  A row's splits are up
// to two runs of partial rows: the own items' and the prefix items'.
struct Row {
  int b, tok, h, n0, n1;
  int64_t row0, row1, step0, step1;
  QF2_DEV int64_t part(int s) const { return s < n0 ? row0 + s * step0 : row1 + (s - n0) * step1; }
};

// the partial rows of output row r, after the attention kernel's end
QF2_DEV Row row_of(const Args& A, int r) {
  Row R;
  const int bt = div_of(A.by_Hq, r);
  R.h = r - bt * A.Hq;
  R.b = div_of(A.by_Sq, bt);
  R.tok = bt - R.b * A.Sq;
  const int Hw = A.Hw, hw = div_of(A.by_G, R.h), g = R.h - hw * A.G, T = A.T;
  const int qt = div_of(A.by_T, R.tok), tr = R.tok - qt * T;
  grid_wait();
  // own run: n0 partial rows, step0 apart, from row0
  R.step0 = (int64_t)A.G * T * A.Nb[0];
  R.step1 = (int64_t)A.G * T * A.Nb[1];
  R.row1 = 0;
  R.n1 = 0;
  if (A.even > 0) {
    const int2 e = A.part_tab[R.b * Hw + hw];
    R.row0 = e.x * R.step0;
    R.n0 = e.y;
  } else {
    R.n0 = A.splits[0];
    R.row0 = (((int64_t)(A.qtiles[0] - 1 - qt) * A.heads[0] + R.b * Hw + hw) * R.n0) * R.step0;
  }
  R.row0 += tr * A.G + g;
  if (A.items1 > 0) {
    const int nb = A.Nb[1], e = R.b / nb, q1 = e * A.qtiles[0] + qt;
    R.n1 = A.splits[1];
    R.row1 = A.part_off1 + (((int64_t)(A.qtiles[1] - 1 - q1) * A.heads[1] + hw) * R.n1) * R.step1 +
             ((R.b - e * nb) * T + tr) * A.G + g;
  }
  return R;
}

QF2_DEV float part_weight(float2 ml, float M) {
  // a NaN sum (its maximum may be -inf: NaN scores leave it) goes on to the output
  return ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : 1.f) : fast_exp2(ml.x - M);
}

template <bool F16>
QF2_DEV void store_row4(const Args& A, const Row& R, int c, float4 a, float l) {
  const bool zero = l == 0.f;
  const float inv = zero ? 0.f : 1.0f / l;
  uint2 w;
  w.x = zero ? 0u : pack16<F16>(a.x * inv, a.y * inv);
  w.y = zero ? 0u : pack16<F16>(a.z * inv, a.w * inv);
  *reinterpret_cast<uint2*>(reinterpret_cast<uint8_t*>(A.out) +
                            2 * (R.b * A.os.b + (int64_t)R.h * A.os.h + R.tok * A.os.s + 4 * c)) = w;
}

// Many rows: one warp per row, 16-byte pieces of a lane (two splits at once where half a warp
// covers the row).  A block a row takes 12 us for 7392 rows of two splits, 64 channels.
template <int D, bool F16>
__global__ void __launch_bounds__(256) mattn_merge_rows_kernel(const __grid_constant__ Args A, int rows) {
  constexpr int C = D / 4, LC = C < 32 ? C : 32, NV = C / LC, NG = 32 / LC;
  const int r = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (r >= rows) return;
  const Row R = row_of(A, r);
  const int ns = R.n0 + R.n1;
  if (ns == 1) return;  // the attention kernel wrote the row
  float M = -INFINITY;
  for (int i = lane; i < ns; i += 32) M = fmaxf(M, A.part_ml[R.part(i)].x);
  for (int d = 16; d; d >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, d));
  const int grp = lane / LC, c = lane - grp * LC;
  const bool on = grp < NG;
  float l = 0.f;
  float4 a[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) a[v] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = 0; s0 < ns; s0 += 32) {
    float w = 0.f;
    if (s0 + lane < ns) {
      const float2 ml = A.part_ml[R.part(s0 + lane)];
      w = part_weight(ml, M);
      l += w * ml.y;
    }
    const int m = min(32, ns - s0);
#pragma unroll 4
    for (int i = 0; i < m; i += NG) {
      const int s = min(i + min(grp, NG - 1), m - 1);  // (past the last split: again, not counted)
      const float ws = __shfl_sync(0xffffffffu, w, s);
      const bool counts = on && i + grp < m && ws != 0.f;  // a split that saw nothing was not written
      const float* o = A.part_o + R.part(s0 + s) * D;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const float4 x = *reinterpret_cast<const float4*>(o + 4 * (v * LC + c));
        if (counts) {
          a[v].x = fmaf(ws, x.x, a[v].x); a[v].y = fmaf(ws, x.y, a[v].y);
          a[v].z = fmaf(ws, x.z, a[v].z); a[v].w = fmaf(ws, x.w, a[v].w);
        }
      }
    }
  }
  for (int d = 16; d; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    if (NG == 2) {
      a[v].x += __shfl_xor_sync(0xffffffffu, a[v].x, 16); a[v].y += __shfl_xor_sync(0xffffffffu, a[v].y, 16);
      a[v].z += __shfl_xor_sync(0xffffffffu, a[v].z, 16); a[v].w += __shfl_xor_sync(0xffffffffu, a[v].w, 16);
    }
    if (grp == 0) store_row4<F16>(A, R, v * LC + c, a[v], l);
  }
}

template <int D, bool F16>
__global__ void __launch_bounds__(128) mattn_merge_kernel(const __grid_constant__ Args A) {
  constexpr int C = D / 4, NG = 128 / C;
  __shared__ float wgt[2 * kMaxSplits];
  __shared__ float4 acc[NG][C];
  const int tid = threadIdx.x;
  const Row R = row_of(A, blockIdx.x);
  const int ns = R.n0 + R.n1;
  if (ns == 1) return;  // the attention kernel wrote the row
  // every warp finds the maximum and the weights by itself (one round of loads, no exchange)
  const int lane = tid & 31;
  float M = -INFINITY;
  for (int i = lane; i < ns; i += 32) M = fmaxf(M, A.part_ml[R.part(i)].x);
  for (int d = 16; d; d >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, d));
  float l = 0.f;
  for (int i = lane; i < ns; i += 32) {
    const float2 ml = A.part_ml[R.part(i)];
    const float w = part_weight(ml, M);
    wgt[i] = w;  // the same from every warp
    l += w * ml.y;
  }
  for (int d = 16; d; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
  __syncwarp();
  const int grp = tid / C, c = tid % C;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  if (grp < NG) {
#pragma unroll 8
    for (int s = grp; s < ns; s += NG) {
      // (loaded whatever its weight, so that the loads do not wait for one another; the row of a
      // split that saw nothing was not written)
      const float w = wgt[s];
      const float4 o = *reinterpret_cast<const float4*>(A.part_o + R.part(s) * D + 4 * c);
      if (w != 0.f) {
        a.x = fmaf(w, o.x, a.x); a.y = fmaf(w, o.y, a.y); a.z = fmaf(w, o.z, a.z); a.w = fmaf(w, o.w, a.w);
      }
    }
    acc[grp][c] = a;
  }
  __syncthreads();
  if (tid < C) {
    for (int k = 1; k < NG; ++k) {
      const float4 o = acc[k][tid];
      a.x += o.x; a.y += o.y; a.z += o.z; a.w += o.w;
    }
    store_row4<F16>(A, R, tid, a, l);
  }
}

// ------------------------------------------------------------------- plan --
struct Plan {
  int form, G, T, Nb[2], qtiles[2], splits[2], ntp, nto, merged, even;
  int64_t items[2];  // CTAs of own and prefix items, splits counted
  bool parts;        // partial rows and a merge
  int64_t rows0;     // partial rows of the own items
  int64_t ids_off, rng_off, qrng_off, order_off, tab_off, ml_off, o_off, bytes;
};

// What of the mask the host knows: the window, the first query's position among all keys, whether
// scores are capped or biased, and whether batch elements may see unlike numbers of keys.
struct Known {
  double left, right, off;  // left, right < 0: open
  bool score, ragged, table;
};

// key tiles that an item of R consecutive tokens sees: the mean of eight items along the queries
static double seen_tiles(const Known& m, int64_t Sq, double keys, double R) {
  double sum = 0.0;
  for (int i = 0; i < 8; ++i) {
    const double c = m.off + (i + 0.5) / 8.0 * (double)Sq;
    const double lo = m.left < 0 ? 0.0 : std::max(0.0, c - 0.5 * R - m.left);
    const double hi = m.right < 0 ? keys : std::min(keys, c + 0.5 * R + m.right);
    sum += std::max(0.0, hi - lo) / kBlk + (lo > 0.0 ? 0.5 : 0.0);  // (a band begins inside a tile)
  }
  return std::max(1.0, sum / 8.0);
}

static int make_plan(Plan* p, int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t Skv, int64_t P, int64_t D,
                     int id_words, const Known& known) {
  if (D != 64 && D != 96 && D != 128 && D != 256) return QF2_ERR_SHAPE;
  if (B < 0 || Sq < 0 || Skv < 0 || P < 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv) return QF2_ERR_SHAPE;
  if (B > 65535 || Hq > 65535 || Sq > (1 << 20)) return QF2_ERR_SHAPE;
  const int64_t ntp = (P + kBlk - 1) / kBlk, nto = (Skv + kBlk - 1) / kBlk;
  if (P > (1 << 20) || Skv > (1 << 20) || ntp + nto > kMaxTiles) return QF2_ERR_SHAPE;
  *p = Plan{};
  p->ntp = (int)ntp;
  p->nto = (int)nto;
  const int64_t group = Hq / Hkv;
  p->Nb[0] = p->Nb[1] = 1;
  p->splits[0] = p->splits[1] = 1;
  p->merged = 1;
  p->G = 1;
  if (B == 0 || Sq == 0) return QF2_OK;
  int64_t hw = Hq;
  // Pack a group's query heads where that makes fewer tiles.  With a distance table only single
  // tokens and up to 16 rows: a head's rows read it from shared memory, a group's from global
  // memory.  24 / 8 heads of 128, packed against not: 300 tokens, reach 512, 33 and 12 us; 4 x 5
  // tokens on 2000 keys 20 and 25; 16 single tokens on 1000 keys 26 and 41.
  const int64_t tp = group <= kBlk ? std::min<int64_t>(Sq, kBlk / group) : 0;
  if ((!known.table || Sq == 1 || group * Sq <= 16) && group > 1 && tp > 0 && Hkv * ((Sq + tp - 1) / tp) < Hq * ((Sq + kBlk - 1) / kBlk)) {
    p->G = (int)group;
    p->T = (int)tp;
    hw = Hkv;
  } else {
    p->T = (int)std::min<int64_t>(Sq, kBlk);
  }
  p->qtiles[0] = (int)((Sq + p->T - 1) / p->T);
  // Two query tiles per CTA, or one in each of two CTAs per SM, where both fill the SMs.  A pair
  // takes less time over a key tile of both, the small ones start and end under each other and
  // leave fewer rows and keys out of sight: waves of CTAs * (tiles seen * time of one + start and
  // end), fitted in us to 204 shapes of 256 to 4096 tokens, 0.2 % off the better of both in the
  // mean (always pairs: 12 %, never: 3 %).  24 / 8 heads of 128, pair against small: 4 x 4096
  // tokens 758 and 826, causal windows of 300 on them 188 and 157, 16 x 512 tokens 88 and 79,
  // 4 x 384 tokens 24.6 and 14.6.
  const int64_t npair = B * Hq * ((Sq + 2 * kBlk - 1) / (2 * kBlk));
  const bool full = D != 256 && Sq > kBlk && npair >= kSms;
  bool two = full;
  const double x = (double)D / 128.0;
  if (full) {
    const double keys = (double)(P + Skv);
    const double pair = seen_tiles(known, Sq, keys, 2.0 * kBlk) * (1.3 + 0.3 * x + (known.score ? 0.5 : 0.0)) + 4.5 + 2.5 * x;
    const double one = seen_tiles(known, Sq, keys, p->T) * (1.5 + 0.5 * x + (known.score ? 0.6 : 0.0)) + 4.5;
    two = (double)((npair + kSms - 1) / kSms) * pair <=
          (double)((B * hw * p->qtiles[0] + 2 * kSms - 1) / (2 * kSms)) * one;
  }
  if (two) {
    p->form = kPair;
    p->G = 1;
    p->T = kBlk;
    hw = Hq;
    p->qtiles[0] = (int)((Sq + 2 * kBlk - 1) / (2 * kBlk));
  } else {
    // rows of several batch elements share a prefix item where two or more fit a tile
    if (P > 0 && p->T == Sq) {
      const int64_t nb = std::min<int64_t>(B, kBlk / ((int64_t)p->G * p->T));
      if (nb > 1) {
        p->merged = 0;
        p->Nb[1] = (int)nb;
        p->qtiles[1] = (int)((B + nb - 1) / nb);
      }
    }
  }
  const int64_t n0 = B * hw * p->qtiles[0], n1 = hw * p->qtiles[1];
  int64_t t0 = (p->merged ? ntp : 0) + nto;  // key tiles of an own item, or of its window
  const int64_t t1 = p->merged ? 0 : ntp;
  if (known.left >= 0.0 && known.right >= 0.0 && P == 0) {
    const double band = ((double)p->T + known.left + known.right + kBlk - 1) / kBlk + 1.0;
    if (band < (double)t0) t0 = std::max<int64_t>(1, (int64_t)band);
  }
  if (full && !two) p->form = kSmall;
  if (!full) {
    // Too few rows to fill the SMs with pairs.  Two forms and any number of splits of the key
    // tiles: a wave of CTAs costs its longest one (a tile takes its latency, or its CTA's share of
    // the memory's rate; 5 us to start and end); a split also writes and reads fp32 partial rows
    // and launches the merge.  kDeep, one CTA per SM, takes less time over a tile than kSmall, two
    // per SM (1.2 against 1.9 us for 128 rows, 0.9 against 1.2 us for the four copies of up to 32),
    // and kSmall takes twice the items in a wave: 500 tokens of 24 / 8 heads of 128 9.9 us in kDeep
    // and 13.7 us in kSmall, 64 single tokens on 4096 keys 176 and 162 us.  Where it misses most: a
    // second wave of memory-bound tiles is priced too high, so that 16 single tokens on 8192 keys of
    // 12 heads of 64 take one split (84 us in the sweep that it was fitted to, 71 with three), and
    // 4 x 16 tokens on 1000 keys 18 % more than the best.
    const bool few = (int64_t)p->G * p->T <= 32;
    const double rows = (double)B * (double)Sq * (double)Hq;
    double best = 1e30, walk = 0.0;
    for (int form = D == 256 || n1 == 0 ? kDeep : kSmall; form >= (D == 256 ? kDeep : kSmall); --form) {
      const int64_t cap = form == kDeep ? kSms : 2 * kSms;  // CTAs at work at once
      double lat = form == kDeep ? (D == 256 ? 2.5 : few ? 0.5 + 0.4 * x : 1.1 + 0.1 * x)
                                 : few ? 0.85 + 0.35 * x : 1.3 + 0.9 * x;
      if (known.score) lat += form == kDeep ? 0.5 : 0.7;
      for (int64_t n = 1; n <= std::min<int64_t>(std::max<int64_t>(t0, 1), kSms); n += 1 + n / 8) {
        const int64_t len = std::max<int64_t>(1, (t0 + n - 1) / n);
        const int64_t s0 = std::max<int64_t>(1, (t0 + len - 1) / len);
        const int64_t ctas = n0 * s0;
        const double walk0 = (double)len * std::max(lat, 1.5 * x * (double)std::min(ctas, cap) / kSms);
        double c = (double)((ctas + cap - 1) / cap) * (walk0 + 5.0);
        if (s0 > 1) c += 2.5 + rows / 2000.0 + rows * (double)s0 * (double)D * 8.0 / 5.0e6;
        if (c < best) {
          best = c;
          walk = walk0;
          p->form = form;
          p->splits[0] = (int)s0;
        }
      }
    }
    const int64_t cap = p->form == kDeep ? kSms : 2 * kSms;
    // prefix items: as many splits as fill the SMs, of four tiles or more
    if (n1 > 0) p->splits[1] = (int)std::max<int64_t>(1, std::min((t1 + 3) / 4, std::min<int64_t>(cap / n1, kMaxSplits)));
    // One query tile per batch element, on unlike lengths that the device knows: split by the keys
    // each has.  That costs 1.2 us before the first load, and gains where the splits are long.
    if (known.ragged && p->qtiles[0] == 1 && B <= kMaxEven && t0 > 2 && 2 * n0 <= cap && walk > 6.0) {
      p->even = (int)cap;
      p->splits[0] = 1;
    }
  }
  p->items[0] = p->even > 0 ? p->even : n0 * p->splits[0];
  p->items[1] = n1 * p->splits[1];
  if (p->items[0] + p->items[1] > 0x7fffffffll) return QF2_ERR_SHAPE;
  p->parts = p->even > 0 || p->splits[0] > 1 || n1 > 0;
  if (p->parts && B * Sq * Hq > 0x7fffffffll) return QF2_ERR_SHAPE;  // the merge's grid
  const int64_t per = (int64_t)p->G * p->T;
  p->rows0 = p->items[0] * per;
  const int64_t rows = p->rows0 + p->items[1] * per * p->Nb[1];
  int64_t off = 0;
  auto take = [&](bool want, int64_t n) {
    const int64_t at = off;
    if (want) off += (n + 255) & ~255ll;
    return at;
  };
  const bool ids = id_words > 0;
  p->ids_off = take(ids, B * nto * kBlk * 4 * id_words);
  p->rng_off = take(ids, B * nto * 8);
  p->qrng_off = take(ids, B * Sq * 8);
  p->order_off = take(ids, B * 4);
  p->tab_off = take(p->even > 0, B * hw * 8);
  p->ml_off = take(p->parts, rows * 8);
  p->o_off = take(p->parts, rows * D * 4);
  p->bytes = off;
  return QF2_OK;
}

// The plan of a call (a window may change it: what of the mask the host knows).
static int plan_of(Plan* p, const qf2_masked_attn_args& M) {
  const int id_words = M.k_ids == nullptr ? 0 : M.ids_i64 ? 2 : 1;
  // (positions and lengths on the device: taken for the end of the keys, and all of them)
  const double first = (double)M.P + (M.q_offset_mode == QF2_OFFSET_CONST ? (double)M.q_offset : (double)M.Skv - (double)M.Sq);
  const Known known{M.prefix_lens ? -1.0 : (double)M.left, (double)M.right, first, M.slopes || M.bias_table || M.softcap > 0.0,
                    M.kv_lens || M.prefix_lens || M.q_offset_mode == QF2_OFFSET_ARRAY, M.bias_table != nullptr};
  int st = make_plan(p, M.B, M.Hq, M.Hkv, M.Sq, M.Skv, M.P, M.D, id_words, known);
  if (st != QF2_OK) return st;
  if (known.left >= 0.0 && known.right >= 0.0) {
    // the workspace is sized without a window: a plan that would take more gives way to that one's
    Known open = known;
    open.left = open.right = -1.0;
    Plan o;
    st = make_plan(&o, M.B, M.Hq, M.Hkv, M.Sq, M.Skv, M.P, M.D, id_words, open);
    if (st != QF2_OK) return st;
    if (p->bytes > o.bytes) *p = o;
  }
  return QF2_OK;
}

static bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// strides {batch, head, seq}; a dimension of one element has no stride to speak of
static int check_strides(const int64_t* st, int64_t B, int64_t H, int64_t S) {
  const int64_t n[3] = {B, H, S};
  for (int i = 0; i < 3; ++i)
    if (n[i] > 1 && (st[i] % 8 || st[i] <= 0 || st[i] >= (1ll << 38))) return QF2_ERR_ALIGN;
  return QF2_OK;
}

// rows of D channels; dims (D, d1, d2, d3) with element strides
static bool make_map(CUtensorMap* m, const void* base, int64_t D, const int64_t n[3], const int64_t st[3],
                     const uint32_t box[3], bool f16) {
  const uint64_t dims[4] = {(uint64_t)D, (uint64_t)n[0], (uint64_t)n[1], (uint64_t)n[2]};
  uint64_t strides[3];
  for (int i = 0; i < 3; ++i) strides[i] = n[i] > 1 ? (uint64_t)st[i] * 2 : (uint64_t)D * 2;
  const uint32_t bx[4] = {64, box[0], box[1], box[2]};
  return qf2_make_tmap_4d(m, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, base, dims,
                          strides, bx);
}

template <bool F16>
static cudaError_t launch_merge(const Args& a, int64_t D, int64_t rows, cudaStream_t s) {
  auto kern = D == 64 ? mattn_merge_kernel<64, F16>
                      : D == 96 ? mattn_merge_kernel<96, F16>
                                : D == 128 ? mattn_merge_kernel<128, F16> : mattn_merge_kernel<256, F16>;
  if (rows >= 16 * kSms) {
    auto many = D == 64 ? mattn_merge_rows_kernel<64, F16>
                        : D == 96 ? mattn_merge_rows_kernel<96, F16>
                                  : D == 128 ? mattn_merge_rows_kernel<128, F16> : mattn_merge_rows_kernel<256, F16>;
    return launch_after(many, dim3((unsigned)((rows + 7) / 8)), 256, 0, s, true, a, (int)rows);
  }
  return launch_after(kern, dim3((unsigned)rows), 128, 0, s, true, a);
}

}  // namespace mattn
}  // namespace qf2

using namespace qf2::mattn;

extern "C" int64_t qf2_masked_attn_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t Skv,
                                                   int64_t P, int64_t D, int with_ids) {
  if (with_ids < 0 || with_ids > 2) return QF2_ERR_ARG;
  // the most that any mask's plan takes (with pairs or without them no rows are split)
  int64_t bytes = 0;
  for (int i = 0; i < 8; ++i) {
    Plan p;
    const int st = make_plan(&p, B, Hq, Hkv, Sq, Skv, P, D, with_ids, Known{-1.0, -1.0, 0.0, (i & 1) != 0, (i & 2) != 0, (i & 4) != 0});
    if (st != QF2_OK) return st;
    bytes = std::max(bytes, p.bytes);
  }
  return bytes;
}

extern "C" int qf2_masked_attn_plan(const qf2_masked_attn_args* args, int64_t* plan) {
  if (!args || !plan) return QF2_ERR_ARG;
  Plan p;
  const int st = plan_of(&p, *args);
  if (st != QF2_OK) return st;
  const int64_t v[8] = {p.form, p.G, p.T, p.splits[0], p.even, p.items[1] > 0 ? p.Nb[1] : 0, p.splits[1], p.bytes};
  for (int i = 0; i < 8; ++i) plan[i] = v[i];
  return QF2_OK;
}

extern "C" int qf2_masked_attn(const qf2_masked_attn_args* args) {
  if (!args) return QF2_ERR_ARG;
  const qf2_masked_attn_args& M = *args;
  const int64_t B = M.B, Hq = M.Hq, Hkv = M.Hkv, Sq = M.Sq, Skv = M.Skv, P = M.P, D = M.D, dtype = M.dtype;
  if (dtype != QF2_BF16 && dtype != QF2_F16) return QF2_ERR_DTYPE;
  const bool ids = M.k_ids != nullptr;
  const int id_words = !ids ? 0 : M.ids_i64 ? 2 : 1;
  Plan p;
  int st = plan_of(&p, M);
  if (st != QF2_OK) return st;
  if (B == 0 || Sq == 0) return QF2_OK;
  if (!M.q || !M.out) return QF2_ERR_ARG;
  if (Skv > 0 && (!M.k || !M.v)) return QF2_ERR_ARG;
  if (P > 0 && (!M.prefix_k || !M.prefix_v)) return QF2_ERR_ARG;
  if ((M.q_ids != nullptr) != ids || (ids && P > 0)) return QF2_ERR_ARG;
  if (M.q_offset_mode < QF2_OFFSET_CONST || M.q_offset_mode > QF2_OFFSET_END ||
      (M.q_offset_mode == QF2_OFFSET_ARRAY && !M.q_offsets))
    return QF2_ERR_ARG;
  if (M.slopes && M.bias_table) return QF2_ERR_ARG;
  if (M.bias_table && (M.bias_reach < 0 || M.bias_reach > kMaxReach)) return QF2_ERR_SHAPE;
  const double l2e = 1.4426950408889634;
  if (!(M.softcap >= 0.0) || !(M.sm_scale > 0.0) || M.softcap > FLT_MAX || M.sm_scale * l2e > FLT_MAX) return QF2_ERR_ARG;
  if (!al16(M.q) || !al16(M.out) || (Skv > 0 && (!al16(M.k) || !al16(M.v))) ||
      (P > 0 && (!al16(M.prefix_k) || !al16(M.prefix_v))))
    return QF2_ERR_ALIGN;
  st = check_strides(M.q_strides, B, Hq, Sq);
  if (st == QF2_OK) st = check_strides(M.out_strides, B, Hq, Sq);
  if (st == QF2_OK && Skv > 0) st = check_strides(M.k_strides, B, Hkv, Skv);
  if (st == QF2_OK && Skv > 0) st = check_strides(M.v_strides, B, Hkv, Skv);
  const int64_t spk[3] = {0, M.prefix_k_strides[0], M.prefix_k_strides[1]};
  const int64_t spv[3] = {0, M.prefix_v_strides[0], M.prefix_v_strides[1]};
  if (st == QF2_OK && P > 0) st = check_strides(spk, 1, Hkv, P);
  if (st == QF2_OK && P > 0) st = check_strides(spv, 1, Hkv, P);
  if (st != QF2_OK) return st;
  if (p.bytes > 0 && (!M.workspace || M.workspace_bytes < p.bytes || !al16(M.workspace))) return QF2_ERR_WORKSPACE;

  const bool f16 = dtype == QF2_F16;
  Maps m;
  {
    const int64_t n[3] = {Hq, Sq, B}, s[3] = {M.q_strides[1], M.q_strides[2], M.q_strides[0]};
    const uint32_t box[3] = {(uint32_t)p.G, (uint32_t)p.T, 1}, box1[3] = {(uint32_t)p.G, (uint32_t)p.T, (uint32_t)p.Nb[1]};
    if (!make_map(&m.q, M.q, D, n, s, box, f16)) return QF2_ERR_ALIGN;
    const int64_t so[3] = {M.out_strides[1], M.out_strides[2], M.out_strides[0]};
    if (!make_map(&m.o, M.out, D, n, so, box, f16)) return QF2_ERR_ALIGN;
    m.q1 = m.q;
    if (p.Nb[1] > 1 && !make_map(&m.q1, M.q, D, n, s, box1, f16)) return QF2_ERR_ALIGN;
  }
  m.k = m.v = m.pk = m.pv = m.q;  // never loaded through where there are no such keys
  const uint32_t kbox[3] = {(uint32_t)kBlk, 1, 1};
  if (Skv > 0) {
    const int64_t n[3] = {Skv, Hkv, B};
    const int64_t sk[3] = {M.k_strides[2], M.k_strides[1], M.k_strides[0]};
    const int64_t sv[3] = {M.v_strides[2], M.v_strides[1], M.v_strides[0]};
    if (!make_map(&m.k, M.k, D, n, sk, kbox, f16) || !make_map(&m.v, M.v, D, n, sv, kbox, f16)) return QF2_ERR_ALIGN;
  }
  if (P > 0) {
    const int64_t n[3] = {P, Hkv, 1};
    const int64_t sk[3] = {spk[2], spk[1], 0}, sv[3] = {spv[2], spv[1], 0};
    if (!make_map(&m.pk, M.prefix_k, D, n, sk, kbox, f16) || !make_map(&m.pv, M.prefix_v, D, n, sv, kbox, f16))
      return QF2_ERR_ALIGN;
  }

  void* status = nullptr;
  QF2_CUDA_CHECK(cudaGetSymbolAddress(&status, g_status));
  uint8_t* ws = reinterpret_cast<uint8_t*>(M.workspace);
  Args a{};
  a.out = M.out;
  a.os = S3{M.out_strides[0], M.out_strides[1], M.out_strides[2]};
  a.B = (int)B; a.Hq = (int)Hq; a.Hkv = (int)Hkv; a.Sq = (int)Sq; a.Skv = (int)Skv; a.P = (int)P;
  a.ntp = p.ntp; a.nto = p.nto;
  a.G = p.G; a.T = p.T;
  for (int i = 0; i < 2; ++i) { a.Nb[i] = p.Nb[i]; a.qtiles[i] = p.qtiles[i]; a.splits[i] = p.splits[i]; }
  a.Hw = (int)(Hq / p.G);
  a.by_G = qf2::make_div(a.G);
  a.by_T = qf2::make_div(a.T);
  a.by_group = qf2::make_div(Hq / Hkv);
  a.by_Hw = qf2::make_div(a.Hw);
  a.by_tt = qf2::make_div(a.qtiles[0]);
  a.by_Hq = qf2::make_div(Hq);
  a.by_Sq = qf2::make_div(Sq);
  for (int i = 0; i < 2; ++i) {
    a.heads[i] = a.Hw * (i == 0 ? a.B : 1);
    a.by_heads[i] = qf2::make_div(a.heads[i]);
    a.by_splits[i] = qf2::make_div(a.splits[i]);
  }
  a.items1 = (int)p.items[1];
  a.merged = p.merged;
  a.even = p.even;
  if (p.parts) {
    a.part_o = reinterpret_cast<float*>(ws + p.o_off);
    a.part_ml = reinterpret_cast<float2*>(ws + p.ml_off);
    a.part_tab = reinterpret_cast<int2*>(ws + p.tab_off);
    a.part_off1 = p.rows0;
  }
  a.kv_lens = M.kv_lens;
  a.prefix_lens = M.prefix_lens;
  a.q_off = M.q_offsets;
  a.q_off_mode = (int)M.q_offset_mode;
  const int64_t far = 1ll << 29;
  a.q_off_const = (int)std::min(std::max(M.q_offset, -far), far);
  a.left = M.left < 0 ? -1 : (int)std::min(M.left, far);
  a.right = M.right < 0 ? -1 : (int)std::min(M.right, far);
  a.q_ids = reinterpret_cast<const int32_t*>(M.q_ids);
  a.id_words = id_words;
  a.hi_off = B * (int64_t)p.nto * kBlk;
  if (ids) {
    a.k_ids = reinterpret_cast<int32_t*>(ws + p.ids_off);
    a.k_rng = reinterpret_cast<int2*>(ws + p.rng_off);
    a.q_rng = reinterpret_cast<int2*>(ws + p.qrng_off);
    a.order = reinterpret_cast<int*>(ws + p.order_off);
    a.aligned = M.q_ids == M.k_ids && Sq == Skv && M.q_offset_mode == QF2_OFFSET_CONST && M.q_offset == 0;
  }
  a.scale = (float)(M.sm_scale * l2e);
  if (M.softcap > 0.0) {
    a.cap_in = (float)std::min(M.sm_scale / M.softcap, 1e37);  // (finite; every score but zero takes the cap)
    a.cap_out = (float)(M.softcap * l2e);
  }
  a.slopes = M.slopes;
  a.table = M.bias_table;
  a.reach = (int)M.bias_reach;
  a.status = reinterpret_cast<int*>(status);
  a.wait_clocks = g_wait_clocks.load(std::memory_order_relaxed);
  a.skip_kv = g_skip_kv.load(std::memory_order_relaxed);
  const bool score = M.softcap > 0.0 || M.slopes || M.bias_table;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(M.stream);
  if (ids) {
    const int kb = (p.nto + 7) / 8;
    const dim3 grid((unsigned)(kb + (Sq + 1023) / 1024), (unsigned)B);
    auto launch = [&](auto type) {
      using I = decltype(type);
      mattn_ids_kernel<I><<<grid, 1024, 0, s>>>(
          reinterpret_cast<const I*>(M.q_ids), reinterpret_cast<const I*>(M.k_ids), (int)Sq, (int)Skv, p.nto, kb,
          reinterpret_cast<int32_t*>(ws + p.ids_off), a.hi_off, reinterpret_cast<int2*>(ws + p.rng_off),
          reinterpret_cast<int2*>(ws + p.qrng_off), reinterpret_cast<int*>(ws + p.order_off));
    };
    if (M.ids_i64) launch(int64_t{});
    else launch(int32_t{});
    QF2_LAUNCH_CHECK();
  }
  const unsigned grid = (unsigned)(p.items[0] + p.items[1]);
  cudaError_t e;
  if (D == 64) e = launch_d64(m, a, grid, p.form, f16, score, s);
  else if (D == 96) e = launch_d96(m, a, grid, p.form, f16, score, s);
  else if (D == 128) e = launch_d128(m, a, grid, p.form, f16, score, s);
  else e = launch_d256(m, a, grid, p.form, f16, score, s);
  QF2_CUDA_CHECK(e);
  if (p.parts) {
    QF2_CUDA_CHECK(f16 ? launch_merge<true>(a, D, B * Sq * Hq, s) : launch_merge<false>(a, D, B * Sq * Hq, s));
  }
  return QF2_OK;
}

extern "C" int qf2_masked_attn_fault_injection(int64_t wait_limit_us, int skip_kv_tile) {
  // SM clocks per microsecond: the B200's 1965 MHz maximum rounded up
  g_wait_clocks.store(wait_limit_us > 0 ? wait_limit_us * 2000 : qf2::kWaitClocks, std::memory_order_relaxed);
  g_skip_kv.store(skip_kv_tile >= 0 ? skip_kv_tile : -1, std::memory_order_relaxed);
  return QF2_OK;
}

extern "C" int qf2_masked_attn_status(qf2_stream_t stream) {
  void* p = nullptr;
  QF2_CUDA_CHECK(cudaGetSymbolAddress(&p, g_status));
  return qf2_workspace_status(p, stream);
}
