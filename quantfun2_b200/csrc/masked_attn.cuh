// Masked, capped and biased 16-bit attention (sm_100a): the kernel and its launcher,
// compiled per head dim in masked_attn_d*.cu; the entry points are in masked_attn.cu.
//
//   s(i, j) = scale q_i.k_j;  s = cap tanh(s / cap);  s += -slope_h |t_i - j| or
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
// NT = 2 (long queries): the two tiles' scores are single buffers of their own, so one tile's
// softmax runs while the tensor cores work for the other, and K and V feed 256 rows.
// NT = 1 (few query rows, or head dim 256, whose output takes half of tensor memory): the
// scores are double-buffered, so the next Q K^T runs under the softmax.
// A tile's rows are (batch element, token, query head of a group): one row per token, or all
// query heads of a kv head packed side by side, so that single tokens read K and V once.
#pragma once
#include "qf2_common.cuh"

namespace qf2 {
namespace mattn {

constexpr int kBlk = 128;             // rows of a query tile, keys of a key tile
constexpr int kTile = 16384;          // 128 rows x 128 bytes: one swizzle column of 64 channels
constexpr int kMaxTiles = 8192;       // key tiles of a call (2^20 keys)
constexpr int kMaxReach = 1024;       // distance table: 2 * reach + 1 entries
constexpr int kTabPad = 256;          // clamped entries on each side of the table in shared memory
constexpr float kTau = 8.0f;          // log2 units the running maximum may lag behind
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxSplits = 320;     // partial rows of one output row
constexpr int kSms = 148;             // B200; sizes the grids and splits (a count, not a limit)

struct S3 { int64_t b, h, s; };

// NT = 2: three warpgroups, so that registers can move from the first (producer, products,
// two idle warps) to the softmax ones: launched with 168 a thread (384 x 168 = 64512), then
// 128 x 56 + 256 x 224 = 64512.  NT = 1: two warps and four, 255 registers each.
constexpr int threads(int nt) { return nt == 2 ? 384 : 192; }
constexpr int kRegsFew = 56, kRegsSoftmax = 224;


struct Args {
  void* out;
  S3 os;
  int B, Hq, Hkv, Sq, Skv, P;       // own keys, shared prefix keys
  int ntp, nto;                       // key tiles of the prefix and of the own keys
  int group;                          // query heads per kv head
  // rows of a tile: g heads x T tokens x Nb batch elements ([0] own items, [1] prefix items)
  int G, T, Nb[2], qtiles[2], splits[2];
  int items1;                         // CTAs of prefix items (they come first)
  int merged;                         // own items walk the prefix tiles too
  float* part_o;                      // split partials: fp32 rows and (max, sum), or null
  float2* part_ml;
  // mask
  const int32_t* kv_lens;
  const int32_t* prefix_lens;
  const int32_t* q_off;
  int q_off_mode;                     // 0 the constant, 1 the array, 2 the sequence's end
  int q_off_const;
  int left, right;                    // band, < 0 open
  const int32_t* q_ids;
  const int32_t* k_ids;               // padded copy [B][nto * 128] (pad -2)
  const int2* k_rng;                  // [B][nto] least and greatest id of a key tile
  // scores
  float scale;                        // plain: sm_scale * log2 e; else see score_args
  float cap_in, cap_out;              // cap > 0: 2 scale log2e / cap, cap log2e; else 0
  const float* slopes;
  const float* table;                 // [Hq][2 * reach + 1]
  int reach;
  int* status;
};

template <int D, int NT>
struct Smem {
  static constexpr int nb = (D + 63) / 64;            // 64-channel columns
  static constexpr int op = nb * kTile;                // bytes of a 128-row operand
  // ring slots (K and V tiles alternate); every variant stays above half of the SM's shared
  // memory, so one CTA is resident and its 512 TMEM columns are free when it starts
  static constexpr int slots = D == 256 ? 2 : (D == 64 ? 8 : (NT == 2 ? 4 : 5));
  static constexpr int q = 0;
  static constexpr int ring = NT * op;
  static constexpr int tab = ring + slots * op;        // distance table with its pads
  static constexpr int tab_floats = 2 * kMaxReach + 1 + 2 * kTabPad;
  static constexpr int bits = tab + ((tab_floats * 4 + 15) & ~15);
  static constexpr int bars = bits + kMaxTiles / 8;
  static constexpr int nbars = 1 + 2 * slots + 2 + 2 + 2 + 1;
  static constexpr int misc = bars + nbars * 8;
  static constexpr int total = misc + 64;
  static_assert(total <= 227 * 1024, "shared memory");
  static_assert(total > 114 * 1024, "one CTA per SM");
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

// bits [0, n) of a 32-bit word
QF2_DEV uint32_t low_bits(int n) { return n >= 32 ? 0xffffffffu : (n <= 0 ? 0u : (1u << n) - 1u); }

// walks the set bits of the active-tile words (every role walks the same sequence)
struct TileIter {
  const uint32_t* w;
  int word;
  uint32_t rest;
  QF2_DEV void init(const uint32_t* bits, int first_word, uint32_t first_rest) {
    w = bits;
    word = first_word;
    rest = first_rest;
  }
  QF2_DEV int next() {
    while (rest == 0) rest = w[++word];
    const int t = word * 32 + __ffs(rest) - 1;
    rest &= rest - 1;
    return t;
  }
};

// SCORE: scores are capped and / or biased (log2 units before the mask); else the scale is
// folded into the exponent
template <int D, int NT, bool F16, bool SCORE>
__global__ void __launch_bounds__(threads(NT), 1)
    masked_attn_kernel(const __grid_constant__ CUtensorMap tmq, const __grid_constant__ CUtensorMap tmq1,
                       const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv,
                       const __grid_constant__ CUtensorMap tmpk, const __grid_constant__ CUtensorMap tmpv,
                       const __grid_constant__ Args A) {
  using L = Smem<D, NT>;
  constexpr int kThreads = threads(NT);
  constexpr int W0 = NT == 2 ? 4 : 2;  // first softmax warp
  constexpr int NS = L::slots;
  constexpr uint32_t kTmemO = 256;  // S at 0 and 128 (P over its first 64 columns), O from 256
  extern __shared__ __align__(1024) uint8_t smem[];
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
  uint64_t* bar_s = bar_empty + NS;         // [2] scores of query tile t (NT = 2) / buffer j & 1
  uint64_t* bar_p = bar_s + 2;              // [2] probabilities written
  uint64_t* bar_o = bar_p + 2;              // [2] NT = 2: O_t complete; NT = 1: PV of tile j, [j & 1]
  uint64_t* bar_drain = bar_o + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::misc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::misc + 4);
  // rows of the CTA: least first key, greatest end, greatest prefix, least and greatest id
  int* red = reinterpret_cast<int*>(smem + L::misc + 8);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // ------------------------------------------------------------- work item --
  int x = blockIdx.x;
  const int kind = x < A.items1 ? 1 : 0;
  if (!kind) x -= A.items1;
  const int nsplit = A.splits[kind];
  const int split = x % nsplit;
  x /= nsplit;
  const int nq = A.qtiles[kind];
  const int qt = nq - 1 - x % nq;  // the last rows first: a causal mask gives them the most keys
  x /= nq;
  const int Hw = A.Hq / A.G;       // head slots: query heads, or kv heads with their group packed
  const int hw = x % Hw, b_item = x / Hw;
  const int hk = A.G > 1 ? hw : hw / A.group;
  const int T = A.T, Nb = A.Nb[kind], G = A.G;
  int b0 = b_item, tok0 = qt * NT * T;
  if (kind) {  // prefix items: tiles over (batch elements, tokens)
    const int tt = (A.Sq + T - 1) / T;
    b0 = (qt / tt) * Nb;
    tok0 = (qt % tt) * T;
  }
  const int t_lo = kind ? 0 : (A.merged ? 0 : A.ntp);
  const int t_hi = kind ? A.ntp : A.ntp + A.nto;

  if (threadIdx.x == 0) {
    mbar_init(bar_q, 1);
    for (int s = 0; s < NS; ++s) {
      mbar_init(bar_full + s, 1);
      mbar_init(bar_empty + s, 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(bar_s + s, 1);
      mbar_init(bar_p + s, 4);
      mbar_init(bar_o + s, 1);
    }
    mbar_init(bar_drain, 1);
    *abort_flag = 0;
    red[0] = 0x7fffffff; red[1] = 0; red[2] = 0; red[3] = 0x7fffffff; red[4] = -1;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0 && lane == 0) {  // Q is on its way while the masks are worked out
    prefetch_tmap(&tmk);
    prefetch_tmap(&tmv);
    mbar_arrive_expect_tx(bar_q, (uint32_t)(NT * L::nb) * 128u * (uint32_t)(G * T * Nb));
    for (int t = 0; t < NT; ++t)
      for (int c = 0; c < L::nb; ++c)
        tma_load_4d(sQ + t * L::op + c * kTile, kind ? &tmq1 : &tmq, c * 64, G > 1 ? hw * G : hw, tok0 + t * T, b0,
                    bar_q);
  }

  // ------------------------------------------------------------- row masks --
  // this thread's row (softmax warps): position, head, and the keys it sees:
  // [lo, hi) or [0, pre), with the id `id`
  const int tile = NT == 2 ? (warp - W0) >> 2 : 0;
  const int quarter = warp & 3;
  const int row = quarter * 32 + lane;
  int rb = 0, rtok = 0, rh = 0, qpos = 0, lo = 0, hi = 0, pre = 0, id = 0;
  bool exists = false;
  if (warp >= W0) {
    const int g = row % G, xr = row / G;
    rtok = tok0 + tile * T + xr % T;
    rb = b0 + xr / T;
    rh = G > 1 ? hw * G + g : hw;
    exists = xr / T < Nb && rb < A.B && rtok < A.Sq;
    const int bc = min(rb, A.B - 1);
    int len = A.Skv;
    if (A.kv_lens) len = min(max(A.kv_lens[bc], 0), A.Skv);
    int off = A.q_off_const;
    if (A.q_off_mode == 1) off = A.q_off[bc];
    off = min(max(off, -(1 << 29)), 1 << 29);
    if (A.q_off_mode == 2) off = len - A.Sq;
    len += A.P;
    qpos = A.P + off + rtok;
    lo = A.left < 0 ? 0 : max(qpos - A.left, 0);
    hi = A.right < 0 ? len : min(max(qpos + A.right + 1, 0), len);
    if (A.prefix_lens) pre = min(max(A.prefix_lens[bc], 0), len);
    bool sees = exists && (lo < hi || pre > 0);
    if (A.q_ids) {
      id = exists ? A.q_ids[(int64_t)bc * A.Sq + rtok] : -1;
      sees = sees && id >= 0;
    }
    if (!sees) { lo = 0; hi = 0; pre = 0; }
    const int wlo = __reduce_min_sync(0xffffffffu, sees && lo < hi ? lo : 0x7fffffff);
    const int whi = __reduce_max_sync(0xffffffffu, hi);
    const int wpre = __reduce_max_sync(0xffffffffu, pre);
    const int wi0 = __reduce_min_sync(0xffffffffu, sees ? id : 0x7fffffff);
    const int wi1 = __reduce_max_sync(0xffffffffu, sees ? id : -1);
    if (lane == 0) {
      atomicMin(red + 0, wlo);
      atomicMax(red + 1, whi);
      atomicMax(red + 2, wpre);
      atomicMin(red + 3, wi0);
      atomicMax(red + 4, wi1);
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
  __syncthreads();
  const int ulo = red[0], uhi = red[1], upre = red[2], uid0 = red[3], uid1 = red[4];

  // ---------------------------------------------------------- active tiles --
  // position of a key tile's first key and the end of its store
  auto tile_pos = [&](int t) -> int { return t < A.ntp ? t * kBlk : A.P + (t - A.ntp) * kBlk; };
  auto tile_end = [&](int t) -> int { return t < A.ntp ? A.P : 0x7fffffff; };
  const int2* krng = A.k_rng ? A.k_rng + (int64_t)b0 * A.nto : nullptr;
  const int w_lo = t_lo >> 5, w_hi = (t_hi + 31) >> 5;
  for (int w = w_lo + warp; w < w_hi; w += kThreads / 32) {
    const int t = w * 32 + lane;
    bool act = t >= t_lo && t < t_hi;
    if (act) {
      const int p0 = tile_pos(t), p1 = min(p0 + kBlk, tile_end(t));
      act = (p0 < uhi && p1 > ulo) || p0 < upre;
      if (act && krng) {
        const int2 r = krng[t - A.ntp];
        act = r.y >= uid0 && r.x <= uid1;
      }
    }
    const uint32_t word = __ballot_sync(0xffffffffu, act);
    if (lane == 0) bits[w] = word;
  }
  __syncthreads();
  int n = 0;  // tiles of this CTA
  TileIter it;
  {
    int total = 0;
    for (int w = w_lo + lane; w < w_hi; w += 32) total += __popc(bits[w]);
    total = __reduce_add_sync(0xffffffffu, total);
    const int f = (int)((int64_t)total * split / nsplit), e = (int)((int64_t)total * (split + 1) / nsplit);
    n = e - f;
    int skip = f, w = w_lo;
    uint32_t rest = w < w_hi ? bits[w] : 0;
    if (n > 0) {
      while (skip >= __popc(rest)) {
        skip -= __popc(rest);
        rest = bits[++w];
      }
      for (; skip > 0; --skip) rest &= rest - 1;
    }
    it.init(bits, w, rest);
  }

  auto fail = [&](int code) {
    atomicExch(A.status, code);
    *abort_flag = 1;
  };
  auto wwait = [&](uint64_t* bar, uint32_t parity) -> bool {
    const bool w = mbar_wait(bar, parity) && (*abort_flag == 0);
    return __all_sync(0xffffffffu, w);
  };

  if (warp < W0) {
  if constexpr (NT == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsFew));
  if (warp == 0) {
    // ------------------------------------------------------------ producer --
    int issued = 0;
    bool ok = true;
    for (int j = 0; ok && j < n; ++j) {
      const int t = it.next();
      const bool px = t < A.ntp;
      const int y = (px ? t : t - A.ntp) * kBlk;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const int i = 2 * j + kv, s = i % NS;
        if (!wwait(bar_empty + s, ((i / NS) & 1) ^ 1)) {
          if (lane == 0) fail(kDevTimeoutProducer);
          ok = false;
          break;
        }
        if (lane == 0) {
          const CUtensorMap* m = kv ? (px ? &tmpv : &tmv) : (px ? &tmpk : &tmk);
          uint8_t* dst = sR + s * L::op;
          mbar_arrive_expect_tx(bar_full + s, L::op);
          for (int c = 0; c < L::nb; ++c) tma_load_4d(dst + c * kTile, m, c * 64, y, hk, px ? 0 : b0, bar_full + s);
        }
        __syncwarp();
        issued = i + 1;
      }
    }
    // copies in flight land before the CTA ends (Q also where no key tile was active)
    if (lane == 0) {
      mbar_wait(bar_q, 0);
      if (*abort_flag)
        for (int i = issued > NS ? issued - NS : 0; i < issued; ++i) mbar_wait(bar_full + (i % NS), (i / NS) & 1);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ----------------------------------------------------------- products --
    if (n > 0) {
      constexpr uint32_t ab = F16 ? 0u : 1u;
      constexpr uint32_t idesc_qk = make_idesc(1, ab, ab, 0, 0, kBlk, kBlk);  // K-major x K-major
      constexpr uint32_t idesc_pv = make_idesc(1, ab, ab, 0, 1, kBlk, D);     // P x MN-major V
      const uint32_t aQ = smem_u32(sQ), aR = smem_u32(sR);
      auto slot_full = [&](int i) -> bool { return wwait(bar_full + i % NS, (i / NS) & 1); };
      auto issue_qk = [&](int t, int buf, int j) {
        if (lane == 0) {
          const uint32_t q = aQ + t * L::op, k = aR + (2 * j % NS) * L::op;
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t off = (kk >> 2) * kTile + (kk & 3) * 32;
            mma_f16(tmem + buf * kBlk, sdesc_sw128_kmajor(q + off), sdesc_sw128_kmajor(k + off), idesc_qk,
                    kk > 0 ? 1u : 0u);
          }
          tc_commit(bar_s + buf);
        }
        __syncwarp();
      };
      auto issue_pv = [&](int t, int buf, int j) {
        if (lane == 0) {
          const uint32_t v = aR + ((2 * j + 1) % NS) * L::op;
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)  // 16 keys per step: 8 TMEM columns of P, 16 rows of V
            mma_f16_tmem_a(tmem + kTmemO + t * 128, tmem + buf * kBlk + kk * 8,
                           sdesc_sw128_mnmajor(v + kk * 16 * 128, kTile, 1024), idesc_pv, (j > 0 || kk > 0) ? 1u : 0u);
        }
        __syncwarp();
      };
      auto release = [&](int i) {
        if (lane == 0) tc_commit(bar_empty + i % NS);
        __syncwarp();
      };
      // keys that no row of the CTA sees weigh nothing, yet 0 * NaN would reach every row:
      // their V rows are cleared (a cache's unused end, padding, another text)
      auto clear_dead = [&](int t, int j) {
        const int p0 = tile_pos(t), p1 = min(p0 + kBlk, tile_end(t));
        bool all = (p1 <= uhi && p0 >= ulo) || p1 <= upre;
        const int32_t* ids = nullptr;
        if (krng) {
          const int2 r = krng[t - A.ntp];
          all = all && r.x >= uid0 && r.y <= uid1;
          ids = A.k_ids + ((int64_t)b0 * A.nto + (t - A.ntp)) * kBlk;
        }
        if (all) return;
        uint8_t* v = sR + ((2 * j + 1) % NS) * L::op;
        for (int r = lane; r < kBlk; r += 32) {
          const int p = p0 + r;
          bool dead = !((p < uhi && p >= ulo) || p < upre) || p >= p1;
          if (ids) dead = dead || ids[r] < uid0 || ids[r] > uid1;
          if (dead)
            for (int c = 0; c < L::nb; ++c)
              for (int u = 0; u < 8; ++u)
                *reinterpret_cast<uint4*>(v + c * kTile + r * 128 + ((u + lane) & 7) * 16) = make_uint4(0, 0, 0, 0);
        }
        fence_async_smem();
        __syncwarp();
      };
      bool ok = wwait(bar_q, 0) && slot_full(0);
      if (ok) {
        tc_fence_after();
        for (int t = 0; t < NT; ++t) issue_qk(t, t, 0);
        release(0);
      }
      for (int j = 0; ok && j < n; ++j) {
        const int kt = it.next();
        const bool more = j + 1 < n;
        if (NT == 1 && more) {
          // the other buffer's P was read by the PV of tile j - 1, issued before this product
          if (!slot_full(2 * j + 2)) { ok = false; break; }
          tc_fence_after();
          issue_qk(0, (j + 1) & 1, j + 1);
          release(2 * j + 2);
        }
        if (!slot_full(2 * j + 1)) { ok = false; break; }
        clear_dead(kt, j);
        if (NT == 2 && more && !slot_full(2 * j + 2)) { ok = false; break; }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const int buf = NT == 2 ? t : (j & 1);
          if (!wwait(bar_p + buf, NT == 2 ? (j & 1) : ((j >> 1) & 1))) { ok = false; break; }
          tc_fence_after();
          issue_pv(t, buf, j);
          if (NT == 2) {
            if (more) {
              issue_qk(t, t, j + 1);
            } else {
              if (lane == 0) tc_commit(bar_o + t);
              __syncwarp();
            }
          }
        }
        if (!ok) break;
        if (NT == 1) {
          if (lane == 0) tc_commit(bar_o + (j & 1));
          __syncwarp();
        }
        release(2 * j + 1);
        if (NT == 2 && more) release(2 * j + 2);
      }
      if (lane == 0) {
        if (!ok) fail(kDevTimeoutMma);
        tc_commit(bar_drain);
        mbar_wait(bar_drain, 0);
      }
      __syncwarp();
    }
  }
  } else {
    // ------------------------------------------------------------ softmax --
    if constexpr (NT == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const uint32_t tO = tmem + lane_off + kTmemO + tile * 128;
    const bool warp_rows = __any_sync(0xffffffffu, exists);
    // what every / any row of this warp sees (rows that do not exist bound nothing)
    const int a_lo = __reduce_max_sync(0xffffffffu, exists ? lo : 0);
    const int a_hi = __reduce_min_sync(0xffffffffu, exists ? hi : 0x7fffffff);
    const int a_pre = __reduce_min_sync(0xffffffffu, exists ? pre : 0x7fffffff);
    const int s_lo = __reduce_min_sync(0xffffffffu, lo < hi ? lo : 0x7fffffff);
    const int s_hi = __reduce_max_sync(0xffffffffu, hi);
    const int s_pre = __reduce_max_sync(0xffffffffu, pre);
    const bool blind = !(lo < hi || pre > 0);
    const int i_lo = __reduce_min_sync(0xffffffffu, exists && !blind ? id : 0x7fffffff);
    const int i_hi = __reduce_max_sync(0xffffffffu, exists && !blind ? id : -1);
    const bool any_blind = __any_sync(0xffffffffu, exists && blind);
    const int q_lo = __reduce_min_sync(0xffffffffu, qpos), q_hi = __reduce_max_sync(0xffffffffu, qpos);
    float slope2 = 0.f;
    const float* trow = nullptr;
    if constexpr (SCORE) {
      const int rhc = min(rh, A.Hq - 1);
      if (A.slopes) slope2 = A.slopes[rhc] * kLog2e;
      if (A.table && !tab_smem) trow = A.table + (int64_t)rhc * (2 * A.reach + 1);
    }
    float m_run = -INFINITY, l_run = 0.f;
    bool ok = true;
    for (int j = 0; ok && j < n; ++j) {
      const int t = it.next();
      const int buf = NT == 2 ? tile : (j & 1);
      if (!wwait(bar_s + buf, NT == 2 ? (j & 1) : ((j >> 1) & 1))) { ok = false; break; }
      tc_fence_after();
      const uint32_t tS = tmem + lane_off + buf * kBlk;
      const int p0 = tile_pos(t), pend = tile_end(t), p1 = min(p0 + kBlk, pend);
      bool any = warp_rows && ((p0 < s_hi && p1 > s_lo) || p0 < s_pre);
      bool full = p0 + kBlk <= pend && ((p1 <= a_hi && p0 >= a_lo) || p1 <= a_pre) && !any_blind;
      const int32_t* kid = nullptr;
      if (krng) {
        const int2 r = krng[t - A.ntp];
        any = any && r.y >= i_lo && r.x <= i_hi;
        if (!(r.x == r.y && i_lo == i_hi && r.x == i_lo)) {
          full = false;
          kid = A.k_ids + ((int64_t)b0 * A.nto + (t - A.ntp)) * kBlk;
        }
      }
      if (!any) {  // no key of the tile is seen: its weights are zero
        uint32_t z[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) z[i] = 0u;
        tmem_st32(tS, z);
        tmem_st32(tS + 32, z);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_p + buf);
        continue;
      }
      float xs[128];
      {
        uint32_t* sr = reinterpret_cast<uint32_t*>(xs);
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(tS + c * 32, *reinterpret_cast<uint32_t(*)[32]>(sr + c * 32));
        tmem_wait_ld();
      }
      if constexpr (SCORE) {
        if (A.cap_in > 0.f) {
          // cap tanh(s / cap) = cap - 2 cap / (1 + e^(2 s / cap)), to 2^-22 of the cap
#pragma unroll
          for (int i = 0; i < 128; ++i) {
            const float e = fast_exp2(xs[i] * A.cap_in);
            xs[i] = fmaf(-2.f * A.cap_out, fast_rcp(1.f + e), A.cap_out);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 128; ++i) xs[i] *= A.scale;
        }
        if (A.slopes) {
          const float d0 = (float)(qpos - p0);
#pragma unroll
          for (int i = 0; i < 128; ++i) xs[i] = fmaf(-slope2, fabsf(d0 - (float)i), xs[i]);
        }
        if (tab_smem) {
          // distances p0 - q_hi .. p0 + 127 - q_lo of this warp
          if (p0 - q_hi >= A.reach || p0 + kBlk - 1 - q_lo <= -A.reach) {
            const float bv = tab[p0 - q_hi >= A.reach ? 2 * A.reach + kTabPad : kTabPad];
#pragma unroll
            for (int i = 0; i < 128; ++i) xs[i] += bv;
          } else {
            const float* tp = tab + (p0 - qpos + A.reach + kTabPad);
#pragma unroll
            for (int i = 0; i < 128; ++i) xs[i] += tp[i];
          }
        } else if (trow) {
          const int d0 = p0 - qpos, R = A.reach;
#pragma unroll
          for (int i = 0; i < 128; ++i) xs[i] += bias_log2(__ldg(trow + min(max(d0 + i, -R), R) + R));
        }
      }
      if (!full) {
        const int e = min(hi, pend) - p0, f = lo - p0, g = min(pre, pend) - p0;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const uint32_t w = (low_bits(e - c * 32) & ~low_bits(f - c * 32)) | low_bits(g - c * 32);
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (!((w >> i) & 1u)) xs[c * 32 + i] = -INFINITY;
        }
        if (kid) {
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const int4 k4 = *reinterpret_cast<const int4*>(kid + 4 * i);
            if (k4.x != id) xs[4 * i] = -INFINITY;
            if (k4.y != id) xs[4 * i + 1] = -INFINITY;
            if (k4.z != id) xs[4 * i + 2] = -INFINITY;
            if (k4.w != id) xs[4 * i + 3] = -INFINITY;
          }
        }
      }
      float mq[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        float m = fmax3(xs[c * 32], xs[c * 32 + 1], xs[c * 32 + 2]);
#pragma unroll
        for (int i = 3; i < 31; i += 2) m = fmax3(m, xs[c * 32 + i], xs[c * 32 + i + 1]);
        mq[c] = fmaxf(m, xs[c * 32 + 31]);
      }
      float mx = fmaxf(fmaxf(mq[0], mq[1]), fmaxf(mq[2], mq[3]));
      if constexpr (!SCORE) mx *= A.scale;
      const float m_new = fmaxf(m_run, mx);
      // (tile rows that do not exist hold whatever shared memory held: they have no vote)
      const bool rescale = __any_sync(0xffffffffu, exists && m_new > m_run + kTau);
      if (rescale) {
        const float alpha = m_run == -INFINITY ? 0.f : fast_exp2(m_run - m_new);
        m_run = m_new;
        l_run *= alpha;
        if (j > 0) {
          // O holds the tiles before this one against the old maximum.  NT = 2: its last PV
          // was issued before the product whose scores were just read; NT = 1: wait for it
          if (NT == 1 && !wwait(bar_o + ((j - 1) & 1), (uint32_t)(((j - 1) >> 1) & 1))) { ok = false; break; }
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
      float2 rs0 = make_float2(0.f, 0.f), rs1 = make_float2(0.f, 0.f);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t w[32];
#pragma unroll
        for (int q = 0; q < 32; ++q) {
          const float2 xx = make_float2(xs[c * 64 + 2 * q], xs[c * 64 + 2 * q + 1]);
          const float2 e = SCORE ? fadd2(xx, nm) : ffma2(xx, scv, nm);
          const float2 pp = make_float2(fast_exp2(e.x), fast_exp2(e.y));
          if (q & 1) rs1 = fadd2(rs1, pp); else rs0 = fadd2(rs0, pp);
          w[q] = pack16<F16>(pp.x, pp.y);
        }
        tmem_st32(tS + c * 32, w);
      }
      l_run += (rs0.x + rs1.x) + (rs0.y + rs1.y);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_p + buf);
    }
    // ------------------------------------------------------------ epilogue --
    // (the scores of tile n - 1 came after PV n - 3, so the parity names one phase)
    if (ok && n > 0) ok = NT == 2 ? wwait(bar_o + tile, 0u) : wwait(bar_o + ((n - 1) & 1), (uint32_t)(((n - 1) >> 1) & 1));
    if (!ok) fail(kDevTimeoutEpilogue);
    tc_fence_after();
    const bool zero = !ok || n == 0 || l_run == 0.f;  // NaN sums go on to the output
    if (A.part_o != nullptr) {
      const int s = kind ? A.splits[0] + split : split;
      const int64_t R = (int64_t)A.B * A.Sq * A.Hq;
      const int64_t r = (int64_t)s * R + ((int64_t)rb * A.Sq + rtok) * A.Hq + rh;
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
    } else if (warp_rows) {
      const float inv_l = zero ? 0.f : 1.0f / l_run;
      uint8_t* dst = reinterpret_cast<uint8_t*>(A.out) +
                     2 * ((int64_t)rb * A.os.b + (int64_t)rh * A.os.h + (int64_t)rtok * A.os.s);
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        if (ok && n > 0) {
          tmem_ld32(tO + c * 32, o);
          tmem_wait_ld();
        }
        if (exists) {
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            uint32_t w[4];
#pragma unroll
            for (int u = 0; u < 4; ++u)
              w[u] = zero ? 0u
                          : pack16<F16>(__uint_as_float(o[8 * v + 2 * u]) * inv_l,
                                        __uint_as_float(o[8 * v + 2 * u + 1]) * inv_l);
            *reinterpret_cast<uint4*>(dst + c * 64 + v * 16) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

struct Maps { CUtensorMap q, q1, k, v, pk, pv; };

template <int D, int NT, bool F16, bool SCORE>
static cudaError_t launch_one(const Maps& m, const Args& a, unsigned grid, cudaStream_t s) {
  static std::atomic<uint64_t> attr{0};
  auto kern = masked_attn_kernel<D, NT, F16, SCORE>;
  if (NT == 2 && attr.load(std::memory_order_acquire) == 0) {
    // the register split below must fit what the block is launched with: an inc beyond it waits for good
    cudaFuncAttributes fa;
    const cudaError_t r = cudaFuncGetAttributes(&fa, kern);
    if (r != cudaSuccess) return r;
    if (fa.numRegs * threads(2) < 128 * kRegsFew + 256 * kRegsSoftmax) return cudaErrorInvalidConfiguration;
  }
  cudaError_t e = qf2_set_smem_once(kern, Smem<D, NT>::total, &attr);
  if (e != cudaSuccess) return e;
  kern<<<grid, threads(NT), Smem<D, NT>::total, s>>>(m.q, m.q1, m.k, m.v, m.pk, m.pv, a);
  return cudaGetLastError();
}

template <int D, int NT>
static cudaError_t launch_nt(const Maps& m, const Args& a, unsigned grid, bool f16, bool score, cudaStream_t s) {
  if (f16) return score ? launch_one<D, NT, true, true>(m, a, grid, s) : launch_one<D, NT, true, false>(m, a, grid, s);
  return score ? launch_one<D, NT, false, true>(m, a, grid, s) : launch_one<D, NT, false, false>(m, a, grid, s);
}

// One launcher per head dim, each in its own translation unit.
cudaError_t launch_d64(const Maps& m, const Args& a, unsigned grid, int nt, bool f16, bool score, cudaStream_t s);
cudaError_t launch_d96(const Maps& m, const Args& a, unsigned grid, int nt, bool f16, bool score, cudaStream_t s);
cudaError_t launch_d128(const Maps& m, const Args& a, unsigned grid, int nt, bool f16, bool score, cudaStream_t s);
cudaError_t launch_d256(const Maps& m, const Args& a, unsigned grid, int nt, bool f16, bool score, cudaStream_t s);

}  // namespace mattn
}  // namespace qf2
