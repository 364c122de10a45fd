// Rotary positions from token positions and frequencies (sm_100a).
//
// Pair p of a head row at position t turns by theta = t * inv_freq[p]:
//   a' = g (a cos - b sin),  b' = g (b cos + a sin)       (inverse: sin -> -sin)
// with (a, b) = (x[p], x[p + r/2]) (half layout) or (x[2p], x[2p+1]) (interleaved); the
// channels past the r rotated ones are copied.  The angle is taken in turns in 64 bits,
// t * inv_freq / 2pi less its nearest whole number (|t| * inv_freq up to 2^31 keeps the
// rest to 2^-22 of a turn), then sincospi in 32 bits; the rotation runs in 32 bits and is
// rounded once.
//
// Bound by HBM: 2 * elements * size bytes; the sines are made once per token and block in
// shared memory and serve every head (64 pairs of 64-bit work against 32 heads x 128
// channels), so no table of positions is stored or read.  65537 tokens of 32 heads of 128 in
// bf16 take 164.5 us, the rate of a plain copy.
#include "qf2_common.cuh"

namespace qf2 {
namespace rotary {

struct Side {
  const void* x;
  void* y;
  int64_t sb, ss, sh;  // input strides (elements)
  int64_t ob, os, oh;  // output strides
};

struct Args {
  Side q, k;
  int Hq, H;  // q heads, q + k heads
  const void* pos;
  int64_t pos_sb, pos_ss;
  int pos64;
  const double* inv_freq;
  int half;   // rotated pairs
  int D;
  int units;  // units of one head row: rotated ones, then copied ones
  int rot_units;
  Div by_units, by_H, by_half;
  int64_t tokens, S;
  int tok_blk;  // tokens of a block
  float gain;
  float sin_gain;  // -gain for the inverse
};

constexpr int kThreads = 256;
constexpr int kMaxEntries = 2048;  // (token, pair) sines of a block: 16 KB
// tokens of a block, and units a thread takes at once (65537 tokens of 32 heads of 128, bf16):
// 8 and 1 164.5 us (6.53 TB/s), 16 and 1 170, 8 and 2 186, 8 and 4 187: more warps at work beat
// more loads of one
constexpr int kMaxTok = 8;
constexpr int kUnroll = 1;

// V elements per access (16 bytes when the rows allow it, else one element or pair);
// half layout: a rotated unit is V channels of the first half and their V partners
template <typename T, int V, bool HALF>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const Args A) {
  constexpr int PP = HALF ? V : (V >= 2 ? V / 2 : 1);  // pairs of a unit
  __shared__ __align__(16) float2 cs[kMaxEntries];
  __shared__ int64_t base[kMaxTok][4];  // q in, q out, k in, k out offset of each token
  const int64_t t0 = (int64_t)blockIdx.x * A.tok_blk;
  const int nt = (int)min((int64_t)A.tok_blk, A.tokens - t0);
  for (int e = threadIdx.x; e < nt * A.half; e += kThreads) {
    const int tk = div_of(A.by_half, e), p = e - tk * A.half;
    const int64_t n = t0 + tk, b = n / A.S, s = n - b * A.S;
    const int64_t pi = b * A.pos_sb + s * A.pos_ss;
    const double t = A.pos64 ? (double)reinterpret_cast<const int64_t*>(A.pos)[pi]
                             : (double)reinterpret_cast<const int32_t*>(A.pos)[pi];
    const double turns = t * A.inv_freq[p] * 0.15915494309189535;
    const float r = (float)(turns - rint(turns));
    float sn, cn;
    sincospif(2.0f * r, &sn, &cn);
    const int j = p % PP;  // a power of two
    const int at = PP >= 2 ? ((j / 2) * A.rot_units + p / PP) * 2 + (j & 1) : p;
    cs[tk * A.half + at] = make_float2(cn * A.gain, sn * A.sin_gain);
  }
  if (threadIdx.x < nt) {
    const int64_t n = t0 + threadIdx.x, b = n / A.S, s = n - b * A.S;
    base[threadIdx.x][0] = b * A.q.sb + s * A.q.ss;
    base[threadIdx.x][1] = b * A.q.ob + s * A.q.os;
    base[threadIdx.x][2] = b * A.k.sb + s * A.k.ss;
    base[threadIdx.x][3] = b * A.k.ob + s * A.k.os;
  }
  __syncthreads();

  struct alignas(V * sizeof(T)) Vec { T e[V]; };
  const int rows = nt * A.H;
  const int total = rows * A.units;
#pragma unroll kUnroll
  for (int i = blockIdx.y * kThreads + threadIdx.x; i < total; i += kThreads * gridDim.y) {
    const int row = div_of(A.by_units, i), u = i - row * A.units;
    const int tk = div_of(A.by_H, row);
    int h = row - tk * A.H;
    const bool is_q = h < A.Hq;
    h -= is_q ? 0 : A.Hq;
    const T* src = reinterpret_cast<const T*>(is_q ? A.q.x : A.k.x) + base[tk][is_q ? 0 : 2] +
                   (int64_t)h * (is_q ? A.q.sh : A.k.sh);
    T* dst = reinterpret_cast<T*>(is_q ? A.q.y : A.k.y) + base[tk][is_q ? 1 : 3] +
             (int64_t)h * (is_q ? A.q.oh : A.k.oh);
    // the sines of a unit's pairs lie two by two, the units side by side: no bank conflicts
    const float2* f = cs + tk * A.half;
    auto sine = [&](int j) -> float2 { return PP >= 2 ? f[((j / 2) * A.rot_units + u) * 2 + (j & 1)] : f[u]; };
    if (u >= A.rot_units) {
      const int c = 2 * A.half + (u - A.rot_units) * V;
      *reinterpret_cast<Vec*>(dst + c) = *reinterpret_cast<const Vec*>(src + c);
    } else if (HALF) {
      const int p = u * V;
      const Vec a = *reinterpret_cast<const Vec*>(src + p);
      const Vec b = *reinterpret_cast<const Vec*>(src + p + A.half);
      Vec oa, ob;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float2 w = sine(j);
        const float x = to_f32(a.e[j]), y = to_f32(b.e[j]);
        oa.e[j] = from_f32<T>(x * w.x - y * w.y);
        ob.e[j] = from_f32<T>(y * w.x + x * w.y);
      }
      *reinterpret_cast<Vec*>(dst + p) = oa;
      *reinterpret_cast<Vec*>(dst + p + A.half) = ob;
    } else if constexpr (V >= 2) {
      const int c = u * V;
      const Vec a = *reinterpret_cast<const Vec*>(src + c);
      Vec o;
#pragma unroll
      for (int j = 0; j < V / 2; ++j) {
        const float2 w = sine(j);
        const float x = to_f32(a.e[2 * j]), y = to_f32(a.e[2 * j + 1]);
        o.e[2 * j] = from_f32<T>(x * w.x - y * w.y);
        o.e[2 * j + 1] = from_f32<T>(y * w.x + x * w.y);
      }
      *reinterpret_cast<Vec*>(dst + c) = o;
    } else {  // rows off the vector alignment: one interleaved pair of single elements
      const int c = 2 * u;
      const float2 w = cs[tk * A.half + u];
      const float x = to_f32(src[c]), y = to_f32(src[c + 1]);
      dst[c] = from_f32<T>(x * w.x - y * w.y);
      dst[c + 1] = from_f32<T>(y * w.x + x * w.y);
    }
  }
}

template <typename T>
static cudaError_t launch(Args& a, bool half_layout, bool vec, bool copy_rest, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  const int v = vec ? V : 1;
  const int rot = 2 * a.half;
  a.rot_units = half_layout ? a.half / v : (vec ? rot / V : a.half);
  a.units = a.rot_units + (copy_rest ? (a.D - rot) / v : 0);
  // tokens of a block: as many as still leave every SM four blocks (148 SMs), so that a
  // block's sines serve more rows and its loads overlap; few tokens are split over the
  // grid's y instead, every block making its token's sines again
  int tb = kMaxTok;
  while (tb > 1 && (tb * a.half > kMaxEntries || a.tokens < (int64_t)tb * 592)) tb >>= 1;
  a.tok_blk = tb;
  const int64_t blocks = (a.tokens + tb - 1) / tb;
  if (blocks > 0x7fffffffll) return cudaErrorInvalidValue;
  a.by_units = make_div(a.units);
  a.by_H = make_div(a.H);
  a.by_half = make_div(a.half);
  const int64_t per = (int64_t)tb * a.H * a.units;
  int64_t y = 592 / blocks;
  y = y < 1 ? 1 : y;
  const int64_t most = (per + kThreads - 1) / kThreads;
  y = y > most ? most : y;
  const dim3 grid((unsigned)blocks, (unsigned)(y > 65535 ? 65535 : y));
  if (vec) {
    if (half_layout) rotary_kernel<T, V, true><<<grid, kThreads, 0, s>>>(a);
    else rotary_kernel<T, V, false><<<grid, kThreads, 0, s>>>(a);
  } else {
    if (half_layout) rotary_kernel<T, 1, true><<<grid, kThreads, 0, s>>>(a);
    else rotary_kernel<T, 1, false><<<grid, kThreads, 0, s>>>(a);
  }
  return cudaGetLastError();
}

}  // namespace rotary
}  // namespace qf2

using namespace qf2::rotary;

extern "C" int qf2_rotary_apply(const qf2_rotary_args* args) {
  if (!args) return QF2_ERR_ARG;
  const qf2_rotary_args& r = *args;
  const int64_t B = r.B, S = r.S, Hq = r.Hq, Hk = r.Hk, D = r.D, rotary_dim = r.rotary_dim, layout = r.layout,
                dtype = r.dtype;
  if (dtype != QF2_F32 && dtype != QF2_F16 && dtype != QF2_BF16) return QF2_ERR_DTYPE;
  if (layout != QF2_ROTARY_HALF && layout != QF2_ROTARY_INTERLEAVED) return QF2_ERR_ARG;
  if (B < 0 || S < 0 || Hq < 0 || Hk < 0 || D <= 0 || D > 1024) return QF2_ERR_SHAPE;
  if (rotary_dim <= 0 || rotary_dim > D || (rotary_dim & 1)) return QF2_ERR_SHAPE;
  if (Hq > 65535 || Hk > 65535 || (S > 0 && B > (int64_t)(1ll << 34) / S)) return QF2_ERR_SHAPE;
  if (B == 0 || S == 0 || Hq + Hk == 0) return QF2_OK;
  if (!r.positions || !r.inv_freq) return QF2_ERR_ARG;
  if ((Hq > 0 && (!r.xq || !r.xq_out)) || (Hk > 0 && (!r.xk || !r.xk_out))) return QF2_ERR_ARG;
  const int esz = dtype == QF2_F32 ? 4 : 2, V = 16 / esz;
  Args a{};
  bool vec = D % V == 0 && (layout == QF2_ROTARY_HALF ? (rotary_dim / 2) % V == 0 : rotary_dim % V == 0);
  bool in_place = true;
  auto side = [&](Side& d, const void* x, void* y, const int64_t* xs, const int64_t* ys) {
    d = Side{x, y, xs[0], xs[1], xs[2], ys[0], ys[1], ys[2]};
    if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) & 15) vec = false;
    for (int i = 0; i < 3; ++i) {
      if (xs[i] % V || ys[i] % V) vec = false;
      if (xs[i] != ys[i]) in_place = false;
    }
    if (x != y) in_place = false;
  };
  if (Hq > 0) side(a.q, r.xq, r.xq_out, r.xq_strides, r.xq_out_strides);
  if (Hk > 0) side(a.k, r.xk, r.xk_out, r.xk_strides, r.xk_out_strides);
  a.Hq = (int)Hq;
  a.H = (int)(Hq + Hk);
  a.pos = r.positions;
  a.pos_sb = r.pos_strides[0];
  a.pos_ss = r.pos_strides[1];
  a.pos64 = r.pos_is_i64 != 0;
  a.inv_freq = r.inv_freq;
  a.half = (int)(rotary_dim / 2);
  a.D = (int)D;
  a.tokens = B * S;
  a.S = S;
  a.gain = (float)r.gain;
  a.sin_gain = r.inverse ? -a.gain : a.gain;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(r.stream);
  const bool hl = layout == QF2_ROTARY_HALF, rest = !in_place;
  cudaError_t e;
  if (dtype == QF2_F32) e = launch<float>(a, hl, vec, rest, s);
  else if (dtype == QF2_F16) e = launch<__half>(a, hl, vec, rest, s);
  else e = launch<__nv_bfloat16>(a, hl, vec, rest, s);
  QF2_CUDA_CHECK(e);
  return QF2_OK;
}
