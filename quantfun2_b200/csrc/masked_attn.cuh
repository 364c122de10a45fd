// Masked, capped and biased 16-bit attention (sm_100a): the kernel and its launcher,
// compiled per head dim in masked_attn_d*.cu; the entry points are in masked_attn.cu.
//
//   s(i, j) = scale q_i.k_j;  s = cap tanh(s / cap);  s -= slope_h |t_i - j| or
//   s += table_h[clamp(j - t_i, -R, R)];  out_i = sum_seen e^s v_j / sum_seen e^s
//
// for the keys j that the query at position t_i sees (a band, a prefix, a length, an id);
// a row that sees none is zero.  One pass over the keys with the running maximum and sum of
// the softmax: both products on tcgen05 kind::f16, fp32 scores and outputs in tensor
// memory, the probabilities rounded to 16 bits over the scores they came from (their sum is
// taken before that rounding, in fp32).
//
// A CTA holds NT query tiles of 128 rows against a stream of 128-key tiles:
//   warp 0      producer: Q once, then K and V tiles by TMA into a ring of slots
//   warp 1      issues the products: S_t = Q_t K^T, then O_t += P_t V
//   the rest    softmax, one thread per row, four warps per query tile
// Three forms:
//   kPair   many rows that see many keys, NT = 2: one tile's softmax runs while the tensor cores
//           work for the other, and K and V feed 256 rows; all of tensor memory, one CTA per SM
//   kSmall  many rows that see few keys each: half of everything, two CTAs per SM, one of which
//           starts, ends or waits for memory while the other works
//   kDeep   few query rows, and head dim 256 (whose output takes half of tensor
//           memory): one CTA per SM with a deep ring; the scores are double-buffered, so the
//           next Q K^T runs under the softmax
// A tile's rows are (batch element, token, query head of a group): one row per token, or all
// query heads of a kv head packed side by side, so that single tokens read K and V once.
//
// Long queries are bound by one chain per tile (scores read, maximum, 128 exponentials a row,
// probabilities stored, the last of P V, the next Q K^T: 3100 cycles for two tiles of which the
// exponent unit works 2048 and the tensor cores 2100), and by the board's power: 16384 causal
// tokens of 24/8 heads of 128 take 1.31 ms cold (1264 TFLOP/s) and 1.56 ms in a long run, where the
// clock falls to 1.7 GHz.  Single tokens are bound by HBM: 16 elements on 8192 keys of 24
// heads 6.4 TB/s.  Short calls are bound by what a CTA does once: 3 us until the first scores,
// 2.5 us after the last.
#pragma once
#include "qf2_common.cuh"

#include <type_traits>

namespace qf2 {
namespace mattn {

constexpr int kBlk = 128;             // rows of a query tile, keys of a key tile
constexpr int kTile = 16384;          // 128 rows x 128 bytes: one swizzle column of 64 channels
constexpr int kMaxTiles = 8192;       // key tiles of a call (2^20 keys)
constexpr int kMaxReach = 1024;       // distance table: 2 * reach + 1 entries
constexpr int kTabPad = 256;          // clamped entries on each side of the table in shared memory
constexpr float kTau = 8.0f;          // log2 units the running maximum may lag behind
constexpr int kPart = 96;             // keys whose P V starts before the rest's exponentials are done
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxSplits = 320;       // partial rows of one output row
constexpr int kMaxEven = 1024;        // batch elements whose lengths a CTA weighs against each other
constexpr int kIdSpan = 4096;         // ids of a CTA's rows that a bitmap holds
constexpr int kSms = 148;             // B200; sizes the grids and splits (a count, not a limit)

struct S3 { int64_t b, h, s; };

template <int N>
using Int = std::integral_constant<int, N>;

// NT = 2: three warpgroups, so that registers can move from the first (producer, products,
// two idle warps) to the softmax ones: launched with 168 a thread (384 x 168 = 64512), then
// 128 x 88 + 256 x 208 = 64512.  (88: with 56 the product warp kept its descriptors in local
// memory.)  The compiler reports 410 to 500 bytes of spill stores for these kernels, about 350 of
// them with the products left out (the softmax warps, whose 128 scores are all in registers) and
// 70 to 200 with the softmax left out; kDeep with capped or biased scores has 8 to 124, kSmall none.
// Two threads per row, exchanging maxima through shared memory, and a first part of
// the exponentials taken before the maximum is known were both slower (8192 x 8192, 24 heads of
// 128: 734 us; 772; 773), as were 1/8 to 3/8 of the exponentials on the FMA pipe, and half key
// tiles with products and barriers of their own (24 heads of 64: 684 us; 863).
constexpr int threads(int nt) { return nt == 2 ? 384 : 192; }
enum Form { kSmall = 0, kDeep = 1, kPair = 2 };
constexpr int kRegsFew = 88, kRegsSoftmax = 208;

// Key ids of a batch element: out of order; out of order, some beyond 31 bits (compared by both
// words); in order (q_rng holds)
enum IdOrder { kMixed = 0, kMixedWide = 1, kInOrder = 2 };

struct Args {
  void* out;
  S3 os;
  int B, Hq, Hkv, Sq, Skv, P;       // own keys, shared prefix keys
  int ntp, nto;                       // key tiles of the prefix and of the own keys
  // rows of a tile: G heads x T tokens x Nb batch elements ([0] own items, [1] prefix items)
  int G, T, Nb[2], qtiles[2], splits[2];
  int Hw;                             // head slots: query heads, or kv heads with their group packed
  int heads[2];                       // head slots of all batch elements (prefix items: of one)
  // (group: query heads per kv head; tt: query tiles of a batch element)
  Div by_G, by_T, by_group, by_Hw, by_heads[2], by_splits[2], by_tt, by_Hq, by_Sq;
  int items1;                         // CTAs of prefix items (they come first)
  int merged;                         // own items walk the prefix tiles too
  int even;                           // > 0: CTAs of the own items, split by what each has to read
  // split partials: fp32 rows, their (max, sum), and the slots of an item where even > 0
  float* part_o;                      // null: no splits
  float2* part_ml;
  int2* part_tab;
  int64_t part_off1;                  // first row of the prefix items' slots
  // mask
  const int32_t* kv_lens;
  const int32_t* prefix_lens;
  const int32_t* q_off;
  int q_off_mode;                     // 0 the constant, 1 the array, 2 the sequence's end
  int q_off_const;
  int left, right;                    // band, < 0 open
  const int32_t* q_ids;               // [B][Sq][id_words]
  int id_words;                       // 2: 64-bit ids, the low word first
  const int32_t* k_ids;               // padded copy [B][nto * 128] (pad -2); of 64-bit ids the low words
  int64_t hi_off;                     // and the high words so many entries behind them
  const int2* k_rng;                  // [B][nto] least and greatest entry of a key tile's copy
  const int2* q_rng;                  // [B][Sq] keys of the row's id, where they are in order
  const int* order;                   // [B] IdOrder of the key ids
  int aligned;                        // query i is key i: one array of ids, no offset
  // scores
  float scale;                        // sm_scale * log2 e
  float cap_in, cap_out;              // cap > 0: scale / cap, cap log2 e; else 0
  const float* slopes;
  const float* table;                 // [Hq][2 * reach + 1]
  int reach;
  int* status;
  long long wait_clocks;              // bound of each wait (kWaitClocks but in tests of it)
  int skip_kv;                        // key tile of a CTA that is never loaded, for such tests; else -1
};

template <int D, int FORM>
struct Smem {
  static constexpr bool two = FORM == kSmall;           // two CTAs per SM
  static constexpr int nt = FORM == kPair ? 2 : 1;
  static constexpr int nb = (D + 63) / 64;            // 64-channel columns
  static constexpr int op = nb * kTile;                // bytes of a 128-row operand
  // ring slots: K and V tiles alternate
  static constexpr int slots = D == 256 ? 2 : (D == 64 ? (two ? 4 : 8) : (two ? 2 : (FORM == kPair ? 4 : 5)));
  static constexpr int q = 0;                           // Q; the output goes out through it
  static constexpr int ring = nt * op;
  static constexpr int tab = ring + slots * op;        // distance table with its pads
  static constexpr int tab_floats = 2 * kMaxReach + 1 + 2 * kTabPad;
  static constexpr int bits = tab + ((tab_floats * 4 + 15) & ~15);
  static constexpr int bars = bits + kMaxTiles / 8;
  static constexpr int nbars = 1 + 2 * slots + 2 + 4 + 2 + 1;
  static constexpr int misc = bars + nbars * 8;
  static constexpr int idbits = misc + 16 + 8 * 8 * 4;  // ids of the rows, where ids are out of order
  static constexpr int rows = (idbits + kIdSpan / 8 + 15) & ~15;  // what each row sees, where rows are unlike
  static constexpr int total = rows + nt * kBlk * 24;
  // TMEM: 512 columns where one CTA has the SM (no second fits beside it), else 256 each
  static constexpr int cols = two ? 256 : 512;
  static_assert(total <= (two ? 113 : 227) * 1024, "shared memory");
  static_assert(two || total > 114 * 1024, "one CTA per SM");
};

template <bool F16>
QF2_DEV uint32_t pack16(float a, float b) {
  if constexpr (F16) {
    const __half2 t = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&t);
  } else {
    const __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&t);
  }
}

QF2_DEV float fast_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// b * log2 e that stays finite where b is: a table of the type's lowest value still gives a
// row an even softmax (only -infinity hides a key)
QF2_DEV float bias_log2(float b) {
  const float r = b * kLog2e;
  return (isinf(r) && !isinf(b)) ? copysignf(3.402823466e38f, b) : r;
}

// co * tanh(ci x) of two scores by the minimax polynomial of tanh(z) / z in z^2 (Remez exchange,
// |z| <= 3/4: to 1.9e-7 of the cap), on the FMA pipe: the quotient with an exponential and a
// reciprocal takes the exponent unit twice as long as the softmax itself does.
constexpr float kTanhMost = 0.75f;
QF2_DEV float2 cap_poly(float2 x, float2 ci, float2 co) {
  const float2 zero = make_float2(0.f, 0.f);
  const float2 z = ffma2(x, ci, zero), t = ffma2(z, z, zero);
  float2 p = ffma2(t, make_float2(0.0123188357f, 0.0123188357f), make_float2(-0.0492804514f, -0.0492804514f));
  p = ffma2(p, t, make_float2(0.132260918f, 0.132260918f));
  p = ffma2(p, t, make_float2(-0.333230765f, -0.333230765f));
  p = ffma2(p, t, make_float2(0.999997228f, 0.999997228f));
  return ffma2(p, ffma2(z, co, zero), zero);
}

// bits [0, n) of a 32-bit word
QF2_DEV uint32_t low_bits(int n) { return n >= 32 ? 0xffffffffu : (n <= 0 ? 0u : (1u << n) - 1u); }

// The key tiles of a CTA: two runs [a0, a0 + na), [b0, ...) of tile numbers, the last first (a
// bias that falls with the distance has its maximum there, and the running maximum then
// does not move: single tokens on 32768 keys with slopes 92 -> 62 us), or (ids out of order)
// the set bits of words in shared memory; every role walks the same sequence.
struct Tiles {
  int a0, na, b0, j;
  const uint32_t* w;  // null: runs
  int word;
  uint32_t rest;
  QF2_DEV int next() {
    if (w == nullptr) {
      const int i = j--;
      return i < na ? a0 + i : b0 + i - na;
    }
    while (rest == 0) rest = w[++word];
    const int t = word * 32 + __ffs(rest) - 1;
    rest &= rest - 1;
    return t;
  }
};

// What the rows of batch element b see by their lengths and offsets.
struct Span { int off, len, pre; };  // own offset of query 0, end of the keys, prefix (positions)
QF2_DEV Span span_of(const Args& A, int b) {
  Span s;
  int len = A.Skv;
  if (A.kv_lens) len = min(max(A.kv_lens[b], 0), A.Skv);
  int off = A.q_off_const;
  if (A.q_off_mode == 1) off = A.q_off[b];
  off = min(max(off, -(1 << 29)), 1 << 29);
  if (A.q_off_mode == 2) off = len - A.Sq;
  s.len = len + A.P;
  s.off = A.P + off;
  s.pre = A.prefix_lens ? min(max(A.prefix_lens[b], 0), s.len) : 0;
  return s;
}

// SCORE: scores are capped and / or biased (log2 units before the mask); else the scale is
// folded into the exponent
template <int D, int FORM, bool F16, bool SCORE>
__global__ void __launch_bounds__(threads(FORM == kPair ? 2 : 1), FORM == kSmall ? 2 : 1)
    masked_attn_kernel(const __grid_constant__ CUtensorMap tmq, const __grid_constant__ CUtensorMap tmq1,
                       const __grid_constant__ CUtensorMap tmo, const __grid_constant__ CUtensorMap tmk,
                       const __grid_constant__ CUtensorMap tmv,
                       const __grid_constant__ CUtensorMap tmpk, const __grid_constant__ CUtensorMap tmpv,
                       const __grid_constant__ Args A) {
  using L = Smem<D, FORM>;
  constexpr int NT = L::nt;
  constexpr bool DB = FORM == kDeep;   // scores double-buffered
  constexpr int kThreads = threads(NT);
  constexpr int W0 = NT == 2 ? 4 : 2;  // first softmax warp
  constexpr int NS = L::slots;
  // S of tile t (or buffer) at t * 128, P over its first 64 columns; O behind them
  constexpr uint32_t kTmemO = L::two ? 128 : 256;
  extern __shared__ __align__(1024) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // ------------------------------------------------------------- work item --
  if (threadIdx.x == 0) {
    prefetch_tmap(&tmq);
    prefetch_tmap(&tmk);
    prefetch_tmap(&tmv);
  }
  int x = blockIdx.x;
  const int kind = x < A.items1 ? 1 : 0;
  if (!kind) x -= A.items1;
  const int T = A.T, Nb = A.Nb[kind], G = A.G, Hw = A.Hw;
  int nsplit = A.splits[kind], split, qt = 0, hw, b0;
  const int slot = x;
  if (!kind && A.even > 0) {
    // One query tile per batch element, lengths known on the device only: the tiles(b) key tiles
    // of an item are split over ceil(tiles(b) / len) CTAs, len such that all fit the grid.
    auto tiles_of = [&](int b) -> int {
      const Span s = span_of(A, b);
      const int base = A.merged ? 0 : A.P;
      const int l = max(A.left < 0 ? 0 : s.off - A.left, base);
      const int h = A.right < 0 ? s.len : min(s.off + A.Sq + A.right, s.len);
      int n = h > l ? (h - base + kBlk - 1) / kBlk - (l - base) / kBlk : 0;
      const int p = min(s.pre, l);
      if (p > base) n += (p - base + kBlk - 1) / kBlk;
      return max(n, 1);
    };
    const int mine = lane < A.B ? tiles_of(lane) : 0;
    float all = (float)mine;
    for (int b = lane + 32; b < A.B; b += 32) all += (float)tiles_of(b);
    for (int d = 16; d; d >>= 1) all += __shfl_xor_sync(0xffffffffu, all, d);
    // rounded up beyond the sum's own rounding, so that the CTAs never outnumber the grid
    const int len = max((int)(__fdividef(all * (float)Hw, (float)(A.even - Hw * A.B)) * 1.0001f) + 1, 2);
    int before = 0, b = -1, c_b = 1, first = 0;
    for (int bb = 0; bb < A.B && b < 0; bb += 32) {
      const int tl = bb == 0 ? mine : (bb + lane < A.B ? tiles_of(bb + lane) : 0);
      const int c = min((int)((uint32_t)(tl + len - 1) / (uint32_t)len), kMaxSplits);
      int sum = c;
      for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, sum, d);
        if (lane >= d) sum += o;
      }
      const uint32_t hit = __ballot_sync(0xffffffffu, (before + sum) * Hw > x);
      if (hit) {
        const int l = __ffs(hit) - 1;
        b = bb + l;
        c_b = __shfl_sync(0xffffffffu, c, l);
        first = (before + __shfl_sync(0xffffffffu, sum, l) - c_b) * Hw;
      } else {
        before += __shfl_sync(0xffffffffu, sum, 31);
      }
    }
    if (b < 0) return;  // the grid has room for the most that rounding up can take
    b0 = b;
    nsplit = c_b;
    hw = (int)((uint32_t)(x - first) / (uint32_t)nsplit);
    split = x - first - hw * nsplit;
    if (threadIdx.x == 0 && split == 0) A.part_tab[b * Hw + hw] = make_int2(x, nsplit);
  } else {
    const int y = div_of(A.by_splits[kind], x);
    split = x - y * nsplit;
    // the last rows of all heads first: a causal mask gives them the most keys, and the short
    // items fill the end of the grid (a head's rows side by side: 4352 tokens with a prefix 256 against 222 us, 16384 causal 1465
    // against 1385)
    const int z = div_of(A.by_heads[kind], y), w = y - z * A.heads[kind];
    qt = A.qtiles[kind] - 1 - z;
    b0 = div_of(A.by_Hw, w);
    hw = w - b0 * Hw;
  }
  const int hk = G > 1 ? hw : div_of(A.by_group, hw);
  int tok0 = qt * NT * T;
  if (kind) {  // prefix items: tiles over (batch elements, tokens)
    const int e = div_of(A.by_tt, qt);
    b0 = e * Nb;
    tok0 = (qt - e * A.qtiles[0]) * T;
  }
  // 32 rows or fewer: four copies of them, one for each softmax warp with a quarter of every key
  // tile (one warp alone took longer over a tile than its keys take from memory)
  const bool quad = FORM != kPair && G * T * Nb <= 32;
  const int t_lo = kind ? 0 : (A.merged ? 0 : A.ntp);
  const int t_hi = kind ? A.ntp : A.ntp + A.nto;

  if (smem_u32(smem) & 1023) {  // the 128-byte swizzle needs 1024-byte aligned tiles
    if (threadIdx.x == 0) atomicExch(A.status, kDevBadLaunch);
    return;
  }
  uint8_t* sQ = smem + L::q;
  uint8_t* sR = smem + L::ring;
  float* tab = reinterpret_cast<float*>(smem + L::tab);
  uint32_t* bits = reinterpret_cast<uint32_t*>(smem + L::bits);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::bars);
  uint64_t* bar_q = bars;
  uint64_t* bar_full = bars + 1;            // [NS]
  uint64_t* bar_empty = bar_full + NS;      // [NS]
  uint64_t* bar_s = bar_empty + NS;         // [2] scores of query tile t (DB: buffer j & 1)
  uint64_t* bar_p = bar_s + 2;              // [2][2] probabilities written: first kPart keys, all
  uint64_t* bar_o = bar_p + 4;              // [2] O_t complete; DB: PV of key tile j, [j & 1]
  uint64_t* bar_drain = bar_o + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::misc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::misc + 4);
  int* red = reinterpret_cast<int*>(smem + L::misc + 16);  // [softmax warp][8]
  uint32_t* idbits = reinterpret_cast<uint32_t*>(smem + L::idbits);
  int4* row_sees = reinterpret_cast<int4*>(smem + L::rows);  // [row] lo, hi, plo, pre
  int2* row_id = reinterpret_cast<int2*>(row_sees + NT * kBlk);

  grid_launch_dependents();  // the merge may take its places; it waits for this grid's end

  // ---------------------------------------------------------- active tiles --
  // position of a key tile's first key, the end of its store, and the tile of a position
  auto tile_pos = [&](int t) -> int { return t < A.ntp ? t * kBlk : A.P + (t - A.ntp) * kBlk; };
  auto tile_end = [&](int t) -> int { return t < A.ntp ? A.P : 0x7fffffff; };
  auto tile_at = [&](int p) -> int { return p < A.P ? p / kBlk : A.ntp + (p - A.P) / kBlk; };
  // what any row of the CTA sees: [ulo, uhi), [uplo, upre), and (ids out of order) ids uid0 .. uid1
  int ulo = 0x7fffffff, uhi = 0, uplo = 0x7fffffff, upre = 0, uid0 = 0x7fffffff, uid1 = -1;
  Tiles it;
  int n = 0;  // tiles of this CTA
  // the two runs in order, without what they share, and this split's part of them
  auto share = [&](int total) -> int {  // first of the split's tiles (at most 2^13 tiles and kMaxSplits splits)
    n = total;
    if (nsplit == 1) return 0;
    const int f = (int)((uint32_t)(total * split) / (uint32_t)nsplit);
    n = (int)((uint32_t)(total * (split + 1)) / (uint32_t)nsplit) - f;
    return f;
  };
  auto runs = [&]() -> int {
    int a0 = t_lo, a1 = t_lo, c0 = t_lo, c1 = t_lo;
    if (uplo < upre) a0 = max(tile_at(uplo), t_lo), a1 = min(tile_at(upre - 1) + 1, t_hi);
    if (ulo < uhi) c0 = max(tile_at(ulo), t_lo), c1 = min(tile_at(uhi - 1) + 1, t_hi);
    if (a0 >= a1 || (c0 < c1 && c0 < a0)) {
      const int s0 = a0, s1 = a1;
      a0 = c0, a1 = c1, c0 = s0, c1 = s1;
    }
    c0 = max(c0, a1);
    it.a0 = a0;
    it.na = max(a1 - a0, 0);
    it.b0 = c0;
    it.w = nullptr;
    it.word = 0;
    it.rest = 0;
    return it.na + max(c1 - c0, 0);
  };
  // Rows of one batch element without ids are consecutive positions: what they see follows from the
  // first and the last, and the first keys are on their way before the rows are looked at.
  const bool direct = A.q_ids == nullptr && Nb == 1;
  if (direct) {
    const Span s = span_of(A, b0);
    const int first = s.off + tok0, last = s.off + min(tok0 + NT * T, A.Sq) - 1;
    ulo = A.left < 0 ? 0 : max(first - A.left, 0);
    uhi = A.right < 0 ? s.len : min(max(last + A.right + 1, 0), s.len);
    uplo = 0;
    upre = s.pre;
    const int total = runs();
    it.j = share(total) + n - 1;
  }
  // K (kv = 0) or V of key tile t into ring slot i % NS
  auto load_kv = [&](int t, int kv, int i) {
    const bool px = t < A.ntp;
    const int y = (px ? t : t - A.ntp) * kBlk, sl = i % NS;
    if (i / 2 == A.skip_kv) return;
    const CUtensorMap* m = kv ? (px ? &tmpv : &tmv) : (px ? &tmpk : &tmk);
    uint8_t* dst = sR + sl * L::op;
    if (elect_one()) {
      mbar_arrive_expect_tx(bar_full + sl, L::op);
#pragma unroll
      for (int c = 0; c < L::nb; ++c) tma_load_4d(dst + c * kTile, m, c * 64, y, hk, px ? 0 : b0, bar_full + sl);
    }
    __syncwarp();
  };
  int ahead = 0;  // tiles loaded before the others are there
  if (warp == 0) {
    // one barrier a lane (one lane for all: 830 cycles)
    static_assert(L::nbars <= 32, "a barrier a lane");
    if (lane < L::nbars) mbar_init(bars + lane, bars + lane >= bar_p && bars + lane < bar_p + 4 ? 4 : 1);
    fence_mbar_init();
    __syncwarp();
    if (elect_one()) {
      *abort_flag = 0;
      const CUtensorMap* mq = kind ? &tmq1 : &tmq;
      const int h0 = G > 1 ? hw * G : hw;
      mbar_arrive_expect_tx(bar_q, (uint32_t)(NT * L::nb * (quad ? 4 : 1)) * 128u * (uint32_t)(G * T * Nb));
      if (FORM != kPair && quad) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int c = 0; c < L::nb; ++c)
            tma_load_4d(sQ + c * kTile + r * 32 * 128, mq, c * 64, h0, tok0, b0, bar_q);
      } else {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int c = 0; c < L::nb; ++c)
            tma_load_4d(sQ + t * L::op + c * kTile, mq, c * 64, h0, tok0 + t * T, b0, bar_q);
      }
    }
    __syncwarp();
    if (direct && n > 0) {
      const int t = it.next();
      load_kv(t, 0, 0);
      load_kv(t, 1, 1);
      ahead = 1;
    }
  } else if (warp == 1) {
    tmem_alloc(tmem_slot, L::cols);
    tmem_relinquish();
  }

  // ------------------------------------------------------------- row masks --
  // this thread's row (softmax warps): position, head, and the keys it sees: [lo, hi) or
  // [plo, pre), and where ids are out of order only those of its id
  const int tile = NT == 2 ? (warp - W0) >> 2 : 0;
  const int quarter = warp & 3;
  const int row = quad ? lane : quarter * 32 + lane;
  int rb = 0, rtok = 0, rh = 0, qpos = 0, lo = 0, hi = 0, plo = 0, pre = 0, id = 0;
  bool exists = false;
  grid_wait();  // for the kernels that prepared the ids (nothing else is still running)
  const int order = A.q_ids != nullptr ? A.order[b0] : kInOrder;
  const bool by_id = order != kInOrder;
  // what any row of this warp sees
  int s_lo = 0x7fffffff, s_hi = 0, s_plo = 0x7fffffff, s_pre = 0, i_lo = 0x7fffffff, i_hi = -1;
  if (warp >= W0) {
    const int xr = div_of(A.by_G, row), g = row - xr * G;
    // (rows behind the tile's last token go on from it where they are of one batch element: the
    // distance table is indexed by consecutive positions)
    const int xb = Nb > 1 ? div_of(A.by_T, xr) : 0;
    rtok = tok0 + tile * T + xr - xb * T;
    rb = b0 + xb;
    rh = G > 1 ? hw * G + g : hw;
    exists = (Nb > 1 ? xb < Nb : xr < T) && rb < A.B && rtok < A.Sq;
    const int bc = min(rb, A.B - 1);
    const Span s = span_of(A, bc);
    qpos = s.off + rtok;
    lo = A.left < 0 ? 0 : max(qpos - A.left, 0);
    hi = A.right < 0 ? s.len : min(max(qpos + A.right + 1, 0), s.len);
    pre = s.pre;
    bool sees = exists;
    if (A.q_ids && exists) {
      const int64_t i = (int64_t)bc * A.Sq + rtok;
      if (by_id) {
        id = A.q_ids[i * A.id_words];
        sees = id >= 0;
        if (A.id_words == 2) {  // (a wide id among narrow keys has none)
          const int top = A.q_ids[2 * i + 1];
          sees = top == 0 ? order == kMixedWide || id >= 0 : order == kMixedWide && top > 0;
          row_id[tile * kBlk + quarter * 32 + lane].y = top;
        }
      } else {
        const int2 r = A.q_rng[i];
        lo = max(lo, r.x);
        hi = min(hi, r.y);
        plo = r.x;
        pre = min(pre, r.y);
      }
    }
    if (!sees || lo >= hi) lo = hi = 0;
    if (!sees || plo >= pre) plo = pre = 0;
    const bool blind = !(lo < hi || plo < pre);
    const int big = 0x7fffffff;
    // A linear bias counts from the nearest key in sight: a row's weights are the same, and those of
    // keys far from the query (|t - j| beyond 2^20 steps, say) do not drown in the bias's rounding.
    if (SCORE && A.slopes && !blind)
      qpos = min(max(qpos, min(lo < hi ? lo : big, plo < pre ? plo : big)), max(hi, pre) - 1);
    s_lo = __reduce_min_sync(0xffffffffu, lo < hi ? lo : big);
    s_hi = __reduce_max_sync(0xffffffffu, hi);
    s_plo = __reduce_min_sync(0xffffffffu, plo < pre ? plo : big);
    s_pre = __reduce_max_sync(0xffffffffu, pre);
    if (by_id) {
      i_lo = __reduce_min_sync(0xffffffffu, blind ? big : id);
      i_hi = __reduce_max_sync(0xffffffffu, blind ? -1 : id);
    }
    if (!direct && (by_id || !A.aligned)) {
      const int r = tile * kBlk + quarter * 32 + lane;
      row_sees[r] = make_int4(lo, hi, plo, pre);
      row_id[r].x = id;
      if (r < kIdSpan / 32) idbits[r] = 0u;
    }
    if (!direct && lane == 0) {
      int* mine = red + (warp - W0) * 8;
      mine[0] = s_lo, mine[1] = s_hi, mine[2] = s_plo, mine[3] = s_pre, mine[4] = i_lo, mine[5] = i_hi;
    }
  }
  // the head's distance table with clamped pads (log2 units), where the rows of a warp are
  // consecutive positions of one head
  const bool tab_smem = SCORE && A.table != nullptr && G == 1 && Nb == 1;
  if (tab_smem) {
    const int R = A.reach, n = 2 * R + 1;
    const float* src = A.table + (int64_t)hw * n;
    for (int i = threadIdx.x; i < n + 2 * kTabPad; i += kThreads)
      tab[i] = bias_log2(__ldg(src + min(max(i - kTabPad, 0), n - 1)));
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int2* krng = by_id ? A.k_rng + (int64_t)b0 * A.nto : nullptr;
  if (!direct) {
#pragma unroll 1
    for (int w = 0; w < 4 * NT; ++w) {
      ulo = min(ulo, red[w * 8]);
      uhi = max(uhi, red[w * 8 + 1]);
      uplo = min(uplo, red[w * 8 + 2]);
      upre = max(upre, red[w * 8 + 3]);
      uid0 = min(uid0, red[w * 8 + 4]);
      uid1 = max(uid1, red[w * 8 + 5]);
    }
    int total = runs();
    if (!krng) {
      it.j = share(total) + n - 1;
    } else {
      const uint32_t nth = (uint32_t)id - (uint32_t)uid0;
      if (warp >= W0 && (lo < hi || plo < pre) && nth < (uint32_t)kIdSpan) atomicOr(idbits + (nth >> 5), 1u << (nth & 31));
      const int w_lo = t_lo >> 5, w_hi = (t_hi + 31) >> 5;
      const int a1 = it.a0 + it.na, c1 = it.b0 + total - it.na;
      for (int w = w_lo + warp; w < w_hi; w += kThreads / 32) {
        const int t = w * 32 + lane;
        bool act = (t >= it.a0 && t < a1) || (t >= it.b0 && t < c1);
        if (act) {
          const int2 r = krng[t - A.ntp];
          act = r.y >= uid0 && r.x <= uid1;
        }
        const uint32_t word = __ballot_sync(0xffffffffu, act);
        if (lane == 0) bits[w] = word;
      }
      __syncthreads();
      total = 0;
      for (int w = w_lo + lane; w < w_hi; w += 32) total += __popc(bits[w]);
      total = __reduce_add_sync(0xffffffffu, total);
      int skip = share(total), w = w_lo;
      if (n > 0) {
        uint32_t rest = bits[w];
        while (skip >= __popc(rest)) {
          skip -= __popc(rest);
          rest = bits[++w];
        }
        for (; skip > 0; --skip) rest &= rest - 1;
        it.w = bits;
        it.word = w;
        it.rest = rest;
      }
    }
  }

  auto fail = [&](int code) {
    atomicExch(A.status, code);
    *abort_flag = 1;
  };
  // warp-wide bounded wait; the abort flag is looked at only while the barrier is not there
  auto wwait = [&](uint64_t* bar, uint32_t parity) -> bool {
    const uint32_t a = smem_u32(bar);
    if (__all_sync(0xffffffffu, mbar_try_wait(a, parity))) return true;
    const long long t0 = clock64();
    while (true) {
      if (__all_sync(0xffffffffu, mbar_try_wait(a, parity))) return true;
      if (__any_sync(0xffffffffu, *abort_flag != 0 || clock64() - t0 > A.wait_clocks)) return false;
    }
  };

  int issued = 0;  // warp 0: copies into the ring
  if (warp < W0) {
    if constexpr (NT == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsFew));
    if (warp == 0) {
      // ---------------------------------------------------------- producer --
      issued = 2 * ahead;
      bool ok = true;
      for (int j = ahead; ok && j < n; ++j) {
        const int t = it.next();
#pragma unroll 1
        for (int kv = 0; kv < 2; ++kv) {
          const int i = 2 * j + kv, s = i % NS;
          if (!wwait(bar_empty + s, ((i / NS) & 1) ^ 1)) {
            if (lane == 0) fail(kDevTimeoutProducer);
            ok = false;
            break;
          }
          load_kv(t, kv, i);
          issued = i + 1;
        }
      }
      // copies in flight land before the CTA ends (Q also where no key tile was active)
      if (lane == 0) mbar_wait(bar_q, 0, A.wait_clocks);
      __syncwarp();
    } else if (warp == 1 && n > 0) {
      // ---------------------------------------------------------- products --
      constexpr uint32_t ab = F16 ? 0u : 1u;
      constexpr uint32_t idesc_qk = make_idesc(1, ab, ab, 0, 0, kBlk, kBlk);  // K-major x K-major
      constexpr uint32_t idesc_pv = make_idesc(1, ab, ab, 0, 1, kBlk, D);     // P x MN-major V
      const uint32_t aR = smem_u32(sR);
      auto slot_full = [&](int i) -> bool { return wwait(bar_full + i % NS, (i / NS) & 1); };
      // descriptors differ from these in the start address alone (16-byte units in the low bits);
      // one elected lane issues, with the warp converged around it (a branch on lane 0 and
      // descriptors built anew took 100 cycles a product of 64: 946 against 737 us, 8192 x 8192,
      // 24 heads of 128)
      const uint64_t dq0 = sdesc_sw128_kmajor(smem_u32(sQ)), dk0 = sdesc_sw128_kmajor(aR);
      const uint64_t dv0 = sdesc_sw128_mnmajor(aR, kTile, 1024);
      // scores of key tile j for query tile t; the key slot is free after the last tile's
      auto issue_qk = [&](int t, int buf, int j) {
        const int slot = 2 * j % NS;
        const uint64_t q = dq0 + (uint64_t)(t * (L::op >> 4)), k = dk0 + (uint64_t)(slot * (L::op >> 4));
        const uint32_t d = tmem + buf * kBlk;
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t off = ((kk >> 2) * kTile + (kk & 3) * 32) >> 4;
            mma_f16(d, q + off, k + off, idesc_qk, kk > 0 ? 1u : 0u);
          }
          tc_commit(bar_s + buf);
          if (t == NT - 1) tc_commit(bar_empty + slot);
        }
        __syncwarp();
      };
      // 16 keys per step: 8 TMEM columns of P, 16 rows of V
      auto issue_pv = [&](int t, int buf, int j, auto k0, auto k1) {
        const uint64_t v = dv0 + (uint64_t)(((2 * j + 1) % NS) * (L::op >> 4));
        const uint32_t d = tmem + kTmemO + t * 128, pa = tmem + buf * kBlk;
        const uint32_t first = j > 0 ? 1u : 0u;
        if (elect_one()) {
#pragma unroll
          for (int kk = k0; kk < k1; ++kk)
            mma_f16_tmem_a(d, pa + kk * 8, v + (uint64_t)(kk * 128), idesc_pv, kk > 0 ? 1u : first);
          if (k1 == kBlk / 16) {
            if (t == NT - 1) tc_commit(bar_empty + (2 * j + 1) % NS);
            if (DB) tc_commit(bar_o + (j & 1));
            else if (j + 1 == n) tc_commit(bar_o + t);
          }
        }
        __syncwarp();
      };
      // Keys that no row of the CTA sees weigh nothing, yet 0 * NaN would reach every row: their V
      // rows are cleared (a cache's unused end, padding, another text).  These are the keys outside
      // of what bounds all rows' ranges and ids, and between them (`look`)
      //   0  none: ranges that follow on each other, one id
      //   1  those of an id that no row has, by a bitmap: every row sees all keys of its id, or all up
      //      to its own, and the keys behind the tile's first row are its rows
      //   2  any: V is looked through for values that are not finite, and their keys are held
      //      against each row (2 x 4000 tokens of ids out of order 707 -> 1093 us, so not where 1 does)
      int look = 0;
      auto choose_look = [&]() {
        if (direct) return;
        const bool wide = krng && A.order[b0] == kMixedWide, many = krng && (uid0 != uid1 || wide);
        if (A.aligned && !many) return;
        if (many && !wide && (uint32_t)uid1 - (uint32_t)uid0 < (uint32_t)kIdSpan && A.left < 0 &&
            (A.right < 0 || (A.aligned && A.right == 0))) {
          look = 1;
          return;
        }
        if (many) {
          look = 2;
          return;
        }
        // no key is missed between ranges that all hold or touch one key, nor where each touches
        // the next row's
        int lo_m = 0, hi_m = 0x7fffffff, lo_p = 0, hi_p = 0x7fffffff, starts = 0;
        bool apart = false;
#pragma unroll 1
        for (int r = lane; r < (quad ? 32 : NT * kBlk); r += 32) {
          const int4 a = row_sees[r];
          const int2 b = r > 0 ? *reinterpret_cast<const int2*>(row_sees + r - 1) : make_int2(0, 0);
          const bool live = a.x < a.y, before = b.x < b.y;
          if (live) lo_m = max(lo_m, a.x), hi_m = min(hi_m, a.y);
          if (a.z < a.w) lo_p = max(lo_p, a.z), hi_p = min(hi_p, a.w);
          starts += live && !before;
          apart = apart || (live && before && max(a.x, b.x) > min(a.y, b.y));
        }
        const unsigned all = 0xffffffffu;
        if ((__reduce_max_sync(all, lo_m) > __reduce_min_sync(all, hi_m) &&
             (__any_sync(all, apart) || __reduce_add_sync(all, starts) > 1)) ||
            __reduce_max_sync(all, lo_p) > __reduce_min_sync(all, hi_p))
          look = 2;
      };
      auto clear_row = [&](uint8_t* v, int r) {
        for (int c = 0; c < L::nb; ++c)
          for (int u = 0; u < 8; ++u)
            *reinterpret_cast<uint4*>(v + c * kTile + r * 128 + ((u + lane) & 7) * 16) = make_uint4(0, 0, 0, 0);
      };
      auto clear_dead = [&](int t, int j, auto looks) {
        const int p0 = tile_pos(t), p1 = min(p0 + kBlk, tile_end(t));
        bool all = (p1 <= uhi && p0 >= ulo) || (p1 <= upre && p0 >= uplo);
        const int32_t* ids = nullptr;
        if (krng) {
          const int2 r = krng[t - A.ntp];
          all = all && r.x >= uid0 && r.y <= uid1;
          ids = A.k_ids + ((int64_t)b0 * A.nto + (t - A.ntp)) * kBlk;
        }
        if (all && (!decltype(looks)::value || look == 0)) return;
        uint8_t* v = sR + ((2 * j + 1) % NS) * L::op;
        for (int r = lane; r < kBlk; r += 32) {
          const int p = p0 + r;
          bool dead = !((p < uhi && p >= ulo) || (p < upre && p >= uplo)) || p >= p1;
          if (ids) {
            const int id = ids[r];
            dead = dead || id < uid0 || id > uid1;
            if (decltype(looks)::value && look == 1 && !dead) dead = !((idbits[(id - uid0) >> 5] >> ((id - uid0) & 31)) & 1u);
          }
          if (dead) clear_row(v, r);
        }
        if (decltype(looks)::value && look == 2) {
#pragma unroll 1
          for (int r = lane; r < kBlk; r += 32) {
            uint32_t top = 0;  // the sign bits of halves whose exponent is all ones (cleared rows have none)
            constexpr uint32_t kExp = F16 ? 0x7c007c00u : 0x7f807f80u, kOne = F16 ? 0x04000400u : 0x00800080u;
#pragma unroll 1
            for (int c = 0; c < L::nb; ++c)
#pragma unroll
              for (int u = 0; u < 8; ++u) {
                const uint4 w = *reinterpret_cast<const uint4*>(v + c * kTile + r * 128 + ((u + lane) & 7) * 16);
                top |= ((w.x & kExp) + kOne) | ((w.y & kExp) + kOne) | ((w.z & kExp) + kOne) | ((w.w & kExp) + kOne);
              }
            uint32_t odd = __ballot_sync(0xffffffffu, (top & 0x80008000u) != 0);
#pragma unroll 1
            while (odd) {
              const int kl = __ffs(odd) - 1, kr = r - lane + kl;
              odd &= odd - 1;
              bool seen = false;
#pragma unroll 1
              for (int i = lane; i < (quad ? 32 : NT * kBlk); i += 32) {
                const int4 m = row_sees[i];
                bool s = (p0 + kr >= m.x && p0 + kr < m.y) || (p0 + kr >= m.z && p0 + kr < m.w);
                if (ids) {
                  s = s && row_id[i].x == ids[kr];
                  if (A.order[b0] == kMixedWide) s = s && row_id[i].y == ids[A.hi_off + kr];
                }
                seen = seen || s;
              }
              if (!__any_sync(0xffffffffu, seen) && lane == kl) clear_row(v, r);
            }
          }
        }
        fence_async_smem();
        __syncwarp();
      };
      // P of key tile j for query tile t in two parts, each multiplied when it is there
      auto pv_when_ready = [&](int t, int buf, int j) -> bool {
        const uint32_t ph = DB ? ((j >> 1) & 1) : (j & 1);
        if (!wwait(bar_p + 2 * buf, ph)) return false;
        tc_fence_after();
        issue_pv(t, buf, j, Int<0>{}, Int<kPart / 16>{});
        if (!wwait(bar_p + 2 * buf + 1, ph)) return false;
        tc_fence_after();
        issue_pv(t, buf, j, Int<kPart / 16>{}, Int<kBlk / 16>{});
        return true;
      };
      bool ok = wwait(bar_q, 0) && slot_full(0);
      if (ok) {
        tc_fence_after();
        for (int t = 0; t < NT; ++t) issue_qk(t, t, 0);
        choose_look();
      }
      // (kPair: the rare looks have a loop of their own; their registers in the one for all calls cost 3
      // to 6 % of the time.  The other forms have registers left, and gain 1 % by the shorter code.)
      auto steps = [&](auto looks) {
        if constexpr (DB) {
          for (int j = 0; ok && j < n; ++j) {
            if (j + 1 < n) {
              // the other buffer's P was read by the PV of tile j - 1, issued before this product
              if (!slot_full(2 * j + 2)) { ok = false; break; }
              tc_fence_after();
              issue_qk(0, (j + 1) & 1, j + 1);
            }
            if (!slot_full(2 * j + 1)) { ok = false; break; }
            clear_dead(it.next(), j, looks);
            if (!pv_when_ready(0, j & 1, j)) { ok = false; break; }
          }
        } else {
          // One warp for both tiles keeps their softmaxes out of phase, so that they take turns
          // at the exponent unit (a warp each: 795 us).  What the next step needs is waited for
          // between the tiles, while the products issued last still run.
          if (ok) ok = slot_full(1) && (NT == 1 || n < 2 || slot_full(2));
          if (ok) clear_dead(it.next(), 0, looks);
          for (int j = 0; ok && j < n; ++j) {
            const bool more = j + 1 < n;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              if (!pv_when_ready(t, t, j)) { ok = false; break; }
              if (!more) continue;
              if (NT == 1 && !slot_full(2 * j + 2)) { ok = false; break; }
              issue_qk(t, t, j + 1);
              if (t == 0) {
                if (!slot_full(2 * j + 3)) { ok = false; break; }
                clear_dead(it.next(), j + 1, looks);
              } else if (j + 2 < n && !slot_full(2 * j + 4)) {
                ok = false;
                break;
              }
            }
          }
        }
      };
      if (FORM == kPair && look == 0) steps(std::false_type{});
      else steps(std::true_type{});
      if (elect_one()) {
        if (!ok) fail(kDevTimeoutMma);
        tc_commit(bar_drain);
        mbar_wait(bar_drain, 0, A.wait_clocks);
      }
      __syncwarp();
    }
  } else {
    // ------------------------------------------------------------ softmax --
    if constexpr (NT == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const uint32_t tO = tmem + lane_off + kTmemO + tile * 128;
    const bool warp_rows = __any_sync(0xffffffffu, exists);
    // what every row of this warp sees (rows that do not exist bound nothing), and what any does
    const int a_lo = __reduce_max_sync(0xffffffffu, exists ? lo : 0);
    const int a_hi = __reduce_min_sync(0xffffffffu, exists ? hi : 0x7fffffff);
    const int a_plo = __reduce_max_sync(0xffffffffu, exists ? plo : 0);
    const int a_pre = __reduce_min_sync(0xffffffffu, exists ? pre : 0x7fffffff);
    // positions of the warp's rows (with tab_smem also of rows past the last query, whose reads of
    // the table must stay inside it; they follow on)
    const bool counts = exists || tab_smem;
    const int q_lo = __reduce_min_sync(0xffffffffu, counts ? qpos : 0x7fffffff);
    const int q_hi = __reduce_max_sync(0xffffffffu, counts ? qpos : -0x7fffffff);
    float slope2 = 0.f;
    const float* trow = nullptr;
    if constexpr (SCORE) {
      const int rhc = min(rh, A.Hq - 1);
      if (A.slopes) slope2 = A.slopes[rhc] * kLog2e;
      if (A.table && !tab_smem) trow = A.table + (int64_t)rhc * (2 * A.reach + 1);
    }
    float m_run = -INFINITY, l_run = 0.f;
    bool ok = true;
    // KW: keys of a tile that a thread takes, from k0 on
    auto softmax = [&](auto kw, const int k0) {
    constexpr int KW = decltype(kw)::value;
    for (int j = 0; ok && j < n; ++j) {
      const int t = it.next();
      const int buf = DB ? (j & 1) : tile;
      if (!wwait(bar_s + buf, DB ? ((j >> 1) & 1) : (j & 1))) { ok = false; break; }
      tc_fence_after();
      const uint32_t tB = tmem + lane_off + buf * kBlk, tS = tB + k0, tP = tB + k0 / 2;
      const int p0 = tile_pos(t) + k0, pend = tile_end(t), p1 = min(p0 + KW, pend);
      bool any = warp_rows && ((p0 < s_hi && p1 > s_lo) || (p0 < s_pre && p1 > s_plo));
      bool full = p0 + KW <= pend && ((p1 <= a_hi && p0 >= a_lo) || (p1 <= a_pre && p0 >= a_plo));
      const int32_t* kid = nullptr;
      if (krng) {
        const int2 r = krng[t - A.ntp];
        any = any && r.y >= i_lo && r.x <= i_hi;
        if (!(r.x == r.y && i_lo == i_hi && r.x == i_lo) || A.order[b0] == kMixedWide) {
          full = false;
          kid = A.k_ids + ((int64_t)b0 * A.nto + (t - A.ntp)) * kBlk + k0;
        }
      }
      if (!any) {  // no key of the tile is seen: its weights are zero
#pragma unroll
        for (int i = 0; i < 8; ++i) tmem_fill8(tB + 8 * i, 0u);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(bar_p + 2 * buf);
          mbar_arrive(bar_p + 2 * buf + 1);
        }
        continue;
      }
      // The scores, first for the maximum, then for the weights: all in registers, or (kSmall, which
      // has fewer) 64 at a time out of tensor memory twice, where capped, biased or masked ones went
      // back to.  16 x 512 tokens, 24 heads of 128, kSmall: 89 us in registers, 80 in loops of 32,
      // 77 in loops of 64; kPair the other way 1385 us in registers, 1438 in loops (causal 16384).
      constexpr bool kHeld = KW == 32 || FORM != kSmall;
      const bool far = SCORE && A.table != nullptr && (p0 - q_hi >= A.reach || p0 + KW - 1 - q_lo <= -A.reach);
      const int e_hi = min(hi, pend) - p0, e_lo = lo - p0, e_pre = min(pre, pend) - p0, e_plo = plo - p0;
      float mx = -INFINITY;
      // N scores, the first of key c of this thread's, into registers (one load: four of 32 columns,
      // each with its own start, 677 against 641 us, 8192 x 8192 tokens, 24 heads of 64; the maximum
      // of 32 under the next 32's load 722)
      auto load = [&](float* x, auto count, int c) {
        constexpr int N = decltype(count)::value;
        if constexpr (N == 128) tmem_ld128(tS + c, *reinterpret_cast<uint32_t(*)[128]>(x));
        else if constexpr (N == 64) tmem_ld64(tS + c, *reinterpret_cast<uint32_t(*)[64]>(x));
        else tmem_ld32(tS + c, *reinterpret_cast<uint32_t(*)[32]>(x));
        tmem_wait_ld();
      };
      auto prepare = [&](float* x, auto count, int c) {
        constexpr int N = decltype(count)::value;
        if constexpr (SCORE) {
          // the scores in log2 units: capped, then sx times the score plus the bias
          float sx = A.scale;
          const int q0 = p0 + c;  // position of x[0]
          if (A.cap_in > 0.f) {
            float ma[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < N; i += 8)
#pragma unroll
              for (int u = 0; u < 4; ++u) ma[u] = fmax3(ma[u], fabsf(x[i + 2 * u]), fabsf(x[i + 2 * u + 1]));
            const float big = fmaxf(fmaxf(ma[0], ma[1]), fmaxf(ma[2], ma[3]));
            // Each score's formula follows from the score alone.  The vote (over hidden keys too) only
            // spares the exponentials where no score needs them, and decides no bit of a result.
            const float2 ci = make_float2(A.cap_in, A.cap_in), co = make_float2(A.cap_out, A.cap_out);
            if (!__any_sync(0xffffffffu, exists && big * A.cap_in > kTanhMost)) {
#pragma unroll
              for (int i = 0; i < N / 2; ++i) {
                const float2 y = cap_poly(make_float2(x[2 * i], x[2 * i + 1]), ci, co);
                x[2 * i] = y.x;
                x[2 * i + 1] = y.y;
              }
            } else {
              // Beyond the polynomial's range cap tanh(z) = cap - 2 cap / (1 + e^(2 z)), to 2^-22 of the
              // cap; within it a small score beside a great cap would be lost in that.  32 scores at a
              // time out of tensor memory and back: with all of them and both formulas in registers
              // 280 bytes more went to local memory, and calls that never come here took 12 % longer.
              const float c2 = 2.f * kLog2e * A.cap_in;
#pragma unroll 1
              for (int u = 0; u < N; u += 32) {
                float s[32];
                tmem_ld32(tS + c + u, *reinterpret_cast<uint32_t(*)[32]>(s));
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; i += 2) {
                  const float2 y = cap_poly(make_float2(s[i], s[i + 1]), ci, co);
                  const float e0 = fmaf(-2.f * A.cap_out, fast_rcp(1.f + fast_exp2(s[i] * c2)), A.cap_out);
                  const float e1 = fmaf(-2.f * A.cap_out, fast_rcp(1.f + fast_exp2(s[i + 1] * c2)), A.cap_out);
                  s[i] = fabsf(s[i]) * A.cap_in > kTanhMost ? e0 : y.x;
                  s[i + 1] = fabsf(s[i + 1]) * A.cap_in > kTanhMost ? e1 : y.y;
                }
                tmem_st32(tS + c + u, *reinterpret_cast<uint32_t(*)[32]>(s));
              }
              tmem_wait_st();
              load(x, count, c);
            }
            sx = 1.f;
          }
          const float2 sx2 = make_float2(sx, sx);
          if (A.slopes) {
            const float d0 = (float)(qpos - q0);
            if (q_lo - q0 >= N - 1 || q_hi <= q0) {
              // all keys on one side of the warp's queries: the bias is linear in the key
              const float sg = q_hi <= q0 ? -slope2 : slope2;
              const float2 sl = make_float2(sg, sg), bb = make_float2(-sg * d0, -sg * d0);
#pragma unroll
              for (int i = 0; i < N / 2; ++i) {
                const float2 y = ffma2(make_float2(x[2 * i], x[2 * i + 1]), sx2,
                                       ffma2(make_float2((float)(2 * i), (float)(2 * i + 1)), sl, bb));
                x[2 * i] = y.x;
                x[2 * i + 1] = y.y;
              }
            } else {
#pragma unroll
              for (int i = 0; i < N; ++i) x[i] = fmaf(-slope2, fabsf(d0 - (float)i), x[i] * sx);
            }
          } else if (far) {  // all distances of the warp beyond the table's reach
            const int end = p0 - q_hi >= A.reach ? 2 * A.reach : 0;
            const float bv = tab_smem ? tab[end + kTabPad] : bias_log2(__ldg(trow + end));
            const float2 bb = make_float2(bv, bv);
#pragma unroll
            for (int i = 0; i < N / 2; ++i) {
              const float2 y = ffma2(make_float2(x[2 * i], x[2 * i + 1]), sx2, bb);
              x[2 * i] = y.x;
              x[2 * i + 1] = y.y;
            }
          } else if (tab_smem) {
            const float* tp = tab + (q0 - qpos + A.reach + kTabPad);
#pragma unroll
            for (int i = 0; i < N; ++i) x[i] = fmaf(x[i], sx, tp[i]);
          } else if (trow) {
            const int d0 = q0 - qpos, R = A.reach;
#pragma unroll
            for (int i = 0; i < N; ++i)
              x[i] = fmaf(x[i], sx, bias_log2(__ldg(trow + min(max(d0 + i, -R), R) + R)));
          }
        }
        if (!full) {
#pragma unroll
          for (int u = 0; u < N; u += 32) {
            const uint32_t w = (low_bits(e_hi - c - u) & ~low_bits(e_lo - c - u)) |
                               (low_bits(e_pre - c - u) & ~low_bits(e_plo - c - u));
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!((w >> i) & 1u)) x[u + i] = -INFINITY;
          }
          if (kid) {
#pragma unroll
            for (int i = 0; i < N / 4; ++i) {
              const int4 k4 = *reinterpret_cast<const int4*>(kid + c + 4 * i);
              if (k4.x != id) x[4 * i] = -INFINITY;
              if (k4.y != id) x[4 * i + 1] = -INFINITY;
              if (k4.z != id) x[4 * i + 2] = -INFINITY;
              if (k4.w != id) x[4 * i + 3] = -INFINITY;
            }
            if (A.order[b0] == kMixedWide) {
              const int top = exists ? A.q_ids[2 * ((int64_t)rb * A.Sq + rtok) + 1] : -1;
#pragma unroll
              for (int i = 0; i < N / 4; ++i) {
                const int4 k4 = *reinterpret_cast<const int4*>(kid + A.hi_off + c + 4 * i);
                if (k4.x != top) x[4 * i] = -INFINITY;
                if (k4.y != top) x[4 * i + 1] = -INFINITY;
                if (k4.z != top) x[4 * i + 2] = -INFINITY;
                if (k4.w != top) x[4 * i + 3] = -INFINITY;
              }
            }
          }
        }
        if (!kHeld && (SCORE || !full)) {
          tmem_st32(tS + c, *reinterpret_cast<uint32_t(*)[32]>(x));
          tmem_st32(tS + c + 32, *reinterpret_cast<uint32_t(*)[32]>(x + 32));
        }
        float m[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) m[u] = fmax3(x[u], x[u + 8], x[u + 16]);
#pragma unroll
        for (int i = 24; i < N - 8; i += 16)
#pragma unroll
          for (int u = 0; u < 8; ++u) m[u] = fmax3(m[u], x[i + u], x[i + u + 8]);
#pragma unroll
        for (int u = 0; u < 8; u += 2) m[u] = fmax3(m[u], m[u + 1], fmaxf(x[N - 8 + u], x[N - 7 + u]));
        mx = fmax3(fmax3(mx, m[0], m[2]), m[4], m[6]);
      };
      float xs[kHeld ? KW : 64];
      if constexpr (kHeld) {
        load(xs, Int<KW>{}, 0);
        prepare(xs, Int<KW>{}, 0);
      } else {
#pragma unroll 1
        for (int c = 0; c < KW; c += 64) {
          load(xs, Int<64>{}, c);
          prepare(xs, Int<64>{}, c);
        }
      }
      if constexpr (!SCORE) mx *= A.scale;
      const float m_new = fmaxf(m_run, mx);
      // (tile rows that do not exist hold whatever shared memory held: they have no vote)
      const bool rescale = __any_sync(0xffffffffu, exists && m_new > m_run + kTau);
      if constexpr (!kHeld) {
        if (SCORE || !full) tmem_wait_st();
      }
      if (rescale) {
        const float alpha = m_run == -INFINITY ? 0.f : fast_exp2(m_run - m_new);
        m_run = m_new;
        l_run *= alpha;
        if (j > 0) {
          // O holds the tiles before this one against the old maximum; their PV was issued
          // before the product whose scores were just read (DB: the last one is waited for)
          if (DB && !wwait(bar_o + ((j - 1) & 1), (uint32_t)(((j - 1) >> 1) & 1))) { ok = false; break; }
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            tmem_ld32(tO + c * 32, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_st32(tO + c * 32, o);
          }
        }
      }
      const float m_use = m_run == -INFINITY ? 0.f : m_run;
      const float sc = SCORE ? 1.f : A.scale;
      const float2 scv = make_float2(sc, sc), nm = make_float2(-m_use, -m_use);
      float2 rs0 = make_float2(0.f, 0.f), rs1 = rs0, rs2 = rs0, rs3 = rs0;
      // weights 2^(s - m), rounded over the scores (16 columns for 32 keys: behind those read)
      auto weigh = [&](float* x, int c) {
        uint32_t w[16];
#pragma unroll
        for (int q = 0; q < 16; ++q) {
          float2 e = make_float2(x[2 * q], x[2 * q + 1]);
          e = SCORE ? fadd2(e, nm) : ffma2(e, scv, nm);
          e.x = fast_exp2(e.x);
          e.y = fast_exp2(e.y);
          if (kHeld && SCORE) {
            x[2 * q] = e.x;
            x[2 * q + 1] = e.y;
          } else {
            float2& rs = q % 4 == 0 ? rs0 : q % 4 == 1 ? rs1 : q % 4 == 2 ? rs2 : rs3;
            rs = fadd2(rs, e);
          }
          w[q] = pack16<F16>(e.x, e.y);
        }
        if (KW == kBlk && c == kPart) {  // the stores of the first keys have landed meanwhile
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar_p + 2 * buf);
        }
        tmem_st16(tP + c / 2, w);
      };
      if constexpr (kHeld) {
#pragma unroll
        for (int c = 0; c < KW; c += 32) weigh(xs + c, c);
        // (quarters: the other ones' keys weigh nothing in this copy of the rows)
#pragma unroll
        for (int i = 0; i < kBlk / KW; ++i)
          if (KW < kBlk && i * KW != k0) {
            tmem_fill8(tB + i * (KW / 2), 0u);
            tmem_fill8(tB + i * (KW / 2) + 8, 0u);
          }
      } else {
#pragma unroll 1
        for (int c = 0; c < KW; c += 64) {
          load(xs, Int<64>{}, c);
          weigh(xs, c);
          weigh(xs + 32, c + 32);
        }
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (KW < kBlk) mbar_arrive(bar_p + 2 * buf);
        mbar_arrive(bar_p + 2 * buf + 1);
      }
      // the row's sum, while the tensor cores go on (without a cap or a bias it is taken under the
      // exponentials: 1200 against 1190 us with a cap, 678 against 685 us without, 8192 x 8192)
      if constexpr (kHeld && SCORE) {
#pragma unroll
        for (int q = 0; q < KW; q += 8) {
          rs0 = fadd2(rs0, make_float2(xs[q], xs[q + 1]));
          rs1 = fadd2(rs1, make_float2(xs[q + 2], xs[q + 3]));
          rs2 = fadd2(rs2, make_float2(xs[q + 4], xs[q + 5]));
          rs3 = fadd2(rs3, make_float2(xs[q + 6], xs[q + 7]));
        }
      }
      rs0 = fadd2(rs0, rs2);
      rs1 = fadd2(rs1, rs3);
      l_run += (rs0.x + rs1.x) + (rs0.y + rs1.y);
    }
    };
    if (FORM != kPair && quad)
      softmax(Int<FORM == kPair ? kBlk : 32>{}, quarter * 32);
    else
      softmax(Int<kBlk>{}, 0);
    // ------------------------------------------------------------ epilogue --
    // (DB: the scores of tile n - 1 came after PV n - 3, so the parity names one phase)
    if (ok && n > 0) ok = DB ? wwait(bar_o + ((n - 1) & 1), (uint32_t)(((n - 1) >> 1) & 1)) : wwait(bar_o + tile, 0u);
    if (n == 0) ok = wwait(bar_q, 0);  // Q's copy has landed before its memory is written
    if (!ok) fail(kDevTimeoutEpilogue);
    tc_fence_after();
    if (FORM != kPair && quad && n > 0) {
      // the four copies' rows become one, through the memory of Q and the ring (every product and
      // copy is done): M = max m_q, sum_q 2^(m_q - M) (l_q, O_q); then each warp has a quarter of
      // the channels
      constexpr int W = D / 4, pitch = D + 4;
      float* so = reinterpret_cast<float*>(smem);
      float2* sml = reinterpret_cast<float2*>(so + kBlk * pitch);
      static_assert(kBlk * pitch * 4 + kBlk * 8 <= L::tab, "rows of four copies");
      if (!ok) l_run = 0.f;
      sml[quarter * 32 + lane] = make_float2(m_run, l_run);
      asm volatile("bar.sync 1, 128;" ::: "memory");
      float M = -INFINITY, l = 0.f, f = 0.f;
#pragma unroll
      for (int q = 0; q < 4; ++q) M = fmaxf(M, sml[q * 32 + lane].x);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float2 e = sml[q * 32 + lane];
        // (a NaN sum whose maximum is -inf goes on to the output)
        const float w = e.y == 0.f ? 0.f : (e.x == -INFINITY ? 1.f : fast_exp2(e.x - M));
        l += w * e.y;
        if (q == quarter) f = w;
      }
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        tmem_ld32(tO + c * 32, o);
        tmem_wait_ld();
        float4* dst = reinterpret_cast<float4*>(so + (quarter * 32 + lane) * pitch + c * 32);
        if (!exists) continue;
#pragma unroll
        for (int v = 0; v < 8; ++v)
          dst[v] = f == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f)
                            : make_float4(__uint_as_float(o[4 * v]) * f, __uint_as_float(o[4 * v + 1]) * f,
                                          __uint_as_float(o[4 * v + 2]) * f, __uint_as_float(o[4 * v + 3]) * f);
      }
      asm volatile("bar.sync 1, 128;" ::: "memory");
      const bool none = !ok || l == 0.f;
      if (exists) {
        const bool parts = A.part_o != nullptr && (nsplit > 1 || A.items1 > 0);
        const int64_t r = (kind ? A.part_off1 : 0) + (int64_t)slot * (G * T * Nb) + row;
        if (parts && quarter == 0) A.part_ml[r] = none ? make_float2(-INFINITY, 0.f) : make_float2(M, l);
        const float inv_l = none ? 0.f : 1.0f / l;
        uint8_t* dst = reinterpret_cast<uint8_t*>(A.out) + 2 * ((int64_t)rb * A.os.b + (int64_t)rh * A.os.h +
                                                                (int64_t)rtok * A.os.s + quarter * W);
#pragma unroll 1
        for (int c = 0; c < W / 8; ++c) {
          float v[8];
#pragma unroll
          for (int u = 0; u < 8; ++u) v[u] = 0.f;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float4* src = reinterpret_cast<const float4*>(so + (q * 32 + lane) * pitch + quarter * W + c * 8);
            const float4 x0 = src[0], x1 = src[1];
            v[0] += x0.x; v[1] += x0.y; v[2] += x0.z; v[3] += x0.w;
            v[4] += x1.x; v[5] += x1.y; v[6] += x1.z; v[7] += x1.w;
          }
          if (parts) {
            float4* po = reinterpret_cast<float4*>(A.part_o + r * D + quarter * W + c * 8);
            if (!none) po[0] = make_float4(v[0], v[1], v[2], v[3]), po[1] = make_float4(v[4], v[5], v[6], v[7]);
          } else {
            uint32_t w[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) w[u] = none ? 0u : pack16<F16>(v[2 * u] * inv_l, v[2 * u + 1] * inv_l);
            *reinterpret_cast<uint4*>(dst + c * 16) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
    }
    const bool joined = FORM != kPair && quad && n > 0;
    const bool zero = !ok || n == 0 || l_run == 0.f;  // NaN sums go on to the output
    if (joined) {
    } else if (A.part_o != nullptr && (nsplit > 1 || A.items1 > 0)) {
      const int64_t r = (kind ? A.part_off1 : 0) + (int64_t)slot * (G * T * Nb) + row;
      if (exists) A.part_ml[r] = zero ? make_float2(-INFINITY, 0.f) : make_float2(m_run, l_run);
      if (warp_rows && n > 0 && ok) {
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          tmem_ld32(tO + c * 32, o);
          tmem_wait_ld();
          if (exists && !zero) {
            uint4* dst = reinterpret_cast<uint4*>(A.part_o + r * D + c * 32);
#pragma unroll
            for (int v = 0; v < 8; ++v) dst[v] = make_uint4(o[4 * v], o[4 * v + 1], o[4 * v + 2], o[4 * v + 3]);
          }
        }
      }
    } else {
      // rows through the Q tile's shared memory (its last product is done) and out by TMA: a
      // thread's own stores of 16 bytes a row took 2200 to 4000 cycles; what lies beyond the
      // tensor is not written
      const float inv_l = zero ? 0.f : 1.0f / l_run;
      uint8_t* so = sQ + tile * L::op + row * 128;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        if (ok && n > 0) {
          tmem_ld32(tO + c * 32, o);
          tmem_wait_ld();
        }
        uint8_t* dst = so + (c >> 1) * kTile;
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          uint32_t w[4];
#pragma unroll
          for (int u = 0; u < 4; ++u)
            w[u] = zero ? 0u
                        : pack16<F16>(__uint_as_float(o[8 * v + 2 * u]) * inv_l,
                                      __uint_as_float(o[8 * v + 2 * u + 1]) * inv_l);
          *reinterpret_cast<uint4*>(dst + ((((c & 1) * 4 + v) ^ (row & 7)) * 16)) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
      fence_async_smem();
      asm volatile("bar.sync %0, 128;" ::"r"(1 + tile) : "memory");
      if (quarter == 0 && lane == 0) {
        for (int c = 0; c < L::nb; ++c)
          tma_store_4d(&tmo, so + c * kTile, c * 64, G > 1 ? hw * G : hw, tok0 + tile * T, b0);
        bulk_commit();
        bulk_wait_read<0>();
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  // (after a wait that gave up nobody has waited for the last copies)
  if (warp == 0 && lane == 0 && *abort_flag)
    for (int i = issued > NS ? issued - NS : 0; i < issued; ++i) mbar_wait(bar_full + (i % NS), (i / NS) & 1, A.wait_clocks);
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, L::cols);
  }
}

// A launch that, with `early`, may begin before the kernel ahead of it in the stream has ended
// (programmatic dependent launch): it reads that kernel's results after grid_wait().
template <typename... P, typename... V>
static cudaError_t launch_after(void (*kern)(P...), dim3 grid, unsigned block, int smem, cudaStream_t s, bool early,
                                const V&... args) {
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = s;
  cfg.attrs = &at;
  cfg.numAttrs = early ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, P(args)...);
}

struct Maps { CUtensorMap q, q1, o, k, v, pk, pv; };

template <int D, int FORM, bool F16, bool SCORE>
static cudaError_t launch_one(const Maps& m, const Args& a, unsigned grid, cudaStream_t s) {
  using L = Smem<D, FORM>;
  static std::atomic<uint64_t> attr{0};
  auto kern = masked_attn_kernel<D, FORM, F16, SCORE>;
  if (FORM == kPair && attr.load(std::memory_order_acquire) == 0) {
    // the register split must fit what the block is launched with: an inc beyond it waits for good
    cudaFuncAttributes fa;
    const cudaError_t r = cudaFuncGetAttributes(&fa, kern);
    if (r != cudaSuccess) return r;
    if (fa.numRegs * threads(2) < 128 * kRegsFew + 256 * kRegsSoftmax) return cudaErrorInvalidConfiguration;
  }
  cudaError_t e = qf2_set_smem_once(kern, L::total, &attr);
  if (e != cudaSuccess) return e;
  return launch_after(kern, grid, threads(L::nt), L::total, s, a.q_ids != nullptr, m.q, m.q1, m.o, m.k, m.v, m.pk, m.pv, a);
}

template <int D, int FORM>
static cudaError_t launch_form(const Maps& m, const Args& a, unsigned grid, bool f16, bool score, cudaStream_t s) {
  if (f16)
    return score ? launch_one<D, FORM, true, true>(m, a, grid, s) : launch_one<D, FORM, true, false>(m, a, grid, s);
  return score ? launch_one<D, FORM, false, true>(m, a, grid, s) : launch_one<D, FORM, false, false>(m, a, grid, s);
}

template <int D>
static cudaError_t launch_dim(const Maps& m, const Args& a, unsigned grid, int form, bool f16, bool score,
                              cudaStream_t s) {
  if (form == kPair) return launch_form<D, kPair>(m, a, grid, f16, score, s);
  if (form == kDeep) return launch_form<D, kDeep>(m, a, grid, f16, score, s);
  return launch_form<D, kSmall>(m, a, grid, f16, score, s);
}

// One launcher per head dim, each in its own translation unit.
cudaError_t launch_d64(const Maps& m, const Args& a, unsigned grid, int form, bool f16, bool score, cudaStream_t s);
cudaError_t launch_d96(const Maps& m, const Args& a, unsigned grid, int form, bool f16, bool score, cudaStream_t s);
cudaError_t launch_d128(const Maps& m, const Args& a, unsigned grid, int form, bool f16, bool score, cudaStream_t s);
cudaError_t launch_d256(const Maps& m, const Args& a, unsigned grid, int form, bool f16, bool score, cudaStream_t s);

}  // namespace mattn
}  // namespace qf2
