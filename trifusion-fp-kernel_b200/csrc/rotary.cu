// Rotary positions of query and key heads at any position, in one launch.
//
//   theta = position * inv_freq[i],  i < R/2
//   (y1, y2) = amplitude * (x1 cos theta - x2 sin theta, x2 cos theta + x1 sin theta)
//
// with the pair (x1, x2) at (i, i + R/2) (half layout) or (2i, 2i + 1)
// (interleaved); elements R.. of each head are copied. Angles are formed in
// turns in FP64 (position * inv_freq / 2 pi, less its nearest integer), so a
// position of 2^31 is off by less than 1e-7 turns; sine and cosine are then FP32
// and the rotation FP32 with one rounding to the type.
//
// Bound by HBM: every element is read and written once. Eight blocks an SM keep enough of
// it on its way (1 x 32768 tokens, 32 + 8 heads of 128: 106 us; 124 us without the bound on
// registers, 102 us at the measured copy rate). A block computes the
// sines and cosines of its tokens once, in shared memory, and all q and k heads
// of those tokens use them.
#include "../../include/trifusion_b200.h"
#include "tf_common.cuh"
#include "tf_host.cuh"

namespace tf {
namespace {

// Quotient by a divisor that the host knows: q = (n * mul) >> 32 is exact for
// n < 2^16 and d < 2^16 with mul = ceil(2^32 / d).
struct FastDiv {
  uint32_t d, mul;
};
FastDiv fast_div(uint32_t d) { return {d, static_cast<uint32_t>((0x100000000ull + d - 1) / d)}; }
__device__ __forceinline__ uint32_t div_by(uint32_t n, const FastDiv& f) { return f.d == 1 ? n : __umulhi(n, f.mul); }

struct RotaryParams {
  const void *q, *k;
  void *qo, *ko;
  int64_t sq[3], sk[3], soq[3], sok[3];  // batch, time, head
  const int64_t* positions;
  int64_t sp[2];
  const double* inv_freq;
  float amplitude;
  int64_t tokens;      // B * T
  int64_t T;
  int tile;            // tokens of a block
  int half;            // R / 2
  int rot_items;       // items of a head that rotate
  int qheads;
  FastDiv items, heads;  // items of a head, q and k heads together
};

constexpr int kThreads = 256;
constexpr int kMaxPairs = 512;  // of one block's tokens
constexpr int kMaxTile = 32;    // tokens of a block

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T x[VEC];
};
__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(bf16 x) { return bf2f(x); }
__device__ __forceinline__ void from_f(float& y, float x) { y = x; }
__device__ __forceinline__ void from_f(bf16& y, float x) { y = __float2bfloat16_rn(x); }

// One item: VEC pairs in the half layout (two vectors), VEC / 2 pairs in the
// interleaved layout (one vector; VEC 1 takes the two elements apart), or one
// vector of the part that does not rotate.
template <typename T, int VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads, 8) rotary_kernel(const __grid_constant__ RotaryParams p) {
  __shared__ float2 cs[kMaxPairs];
  __shared__ int64_t at[kMaxTile][4];  // of a token in q, k and the outputs: 64-bit divisions are for tokens, not items
  const int64_t first = static_cast<int64_t>(blockIdx.x) * p.tile;
  const int ntok = static_cast<int>(min(static_cast<int64_t>(p.tile), p.tokens - first));
  if (threadIdx.x < ntok) {
    const int64_t b = (first + threadIdx.x) / p.T, t = (first + threadIdx.x) - b * p.T;
    at[threadIdx.x][0] = b * p.sq[0] + t * p.sq[1];
    at[threadIdx.x][1] = b * p.sk[0] + t * p.sk[1];
    at[threadIdx.x][2] = b * p.soq[0] + t * p.soq[1];
    at[threadIdx.x][3] = b * p.sok[0] + t * p.sok[1];
  }
  for (int i = threadIdx.x; i < ntok * p.half; i += kThreads) {
    const int tok = i / p.half, pair = i - tok * p.half;
    const uint32_t x = static_cast<uint32_t>(first) + tok, b = x / static_cast<uint32_t>(p.T);
    const int64_t position = p.positions[b * p.sp[0] + (x - b * static_cast<uint32_t>(p.T)) * p.sp[1]];
    double turns = static_cast<double>(position) * (p.inv_freq[pair] * 0.15915494309189533577);
    turns -= rint(turns);
    float s, c;
    sincospif(2.f * static_cast<float>(turns), &s, &c);
    cs[i] = make_float2(c * p.amplitude, s * p.amplitude);
  }
  __syncthreads();
  const int total = ntok * static_cast<int>(p.heads.d * p.items.d);
  for (int idx = threadIdx.x; idx < total; idx += kThreads) {
    const uint32_t row = div_by(idx, p.items), item = idx - row * p.items.d;
    const uint32_t tok = div_by(row, p.heads);
    int head = row - tok * p.heads.d;
    const T* x;
    T* y;
    if (head < p.qheads) {
      x = static_cast<const T*>(p.q) + at[tok][0] + head * p.sq[2];
      y = static_cast<T*>(p.qo) + at[tok][2] + head * p.soq[2];
    } else {
      head -= p.qheads;
      x = static_cast<const T*>(p.k) + at[tok][1] + head * p.sk[2];
      y = static_cast<T*>(p.ko) + at[tok][3] + head * p.sok[2];
    }
    using V = Pack<T, VEC>;
    if (static_cast<int>(item) >= p.rot_items) {  // the part that does not rotate
      const int e = 2 * p.half + (item - p.rot_items) * VEC;
      *reinterpret_cast<V*>(y + e) = *reinterpret_cast<const V*>(x + e);
    } else if (!INTERLEAVED || VEC == 1) {
      constexpr int kPairs = VEC;
      const int e1 = INTERLEAVED ? 2 * item : item * VEC, e2 = INTERLEAVED ? e1 + 1 : e1 + p.half;
      const V a = *reinterpret_cast<const V*>(x + e1), z = *reinterpret_cast<const V*>(x + e2);
      V ya, yz;
      const float2* w = cs + tok * p.half + item * kPairs;
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        const float2 r = w[i];
        const float xa = to_f(a.x[i]), xz = to_f(z.x[i]);
        from_f(ya.x[i], xa * r.x - xz * r.y);
        from_f(yz.x[i], xz * r.x + xa * r.y);
      }
      *reinterpret_cast<V*>(y + e1) = ya;
      *reinterpret_cast<V*>(y + e2) = yz;
    } else {
      constexpr int kPairs = VEC / 2 > 0 ? VEC / 2 : 1;
      const V a = *reinterpret_cast<const V*>(x + item * VEC);
      V ya;
      const float2* w = cs + tok * p.half + item * kPairs;
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        const float2 r = w[i];
        const float xa = to_f(a.x[2 * i]), xz = to_f(a.x[(2 * i + 1) % VEC]);
        from_f(ya.x[2 * i], xa * r.x - xz * r.y);
        from_f(ya.x[(2 * i + 1) % VEC], xz * r.x + xa * r.y);
      }
      *reinterpret_cast<V*>(y + item * VEC) = ya;
    }
  }
}

template <typename T, int VEC>
void launch(const RotaryParams& p, bool interleaved, cudaStream_t stream) {
  const unsigned grid = static_cast<unsigned>((p.tokens + p.tile - 1) / p.tile);
  if (interleaved)
    rotary_kernel<T, VEC, true><<<grid, kThreads, 0, stream>>>(p);
  else
    rotary_kernel<T, VEC, false><<<grid, kThreads, 0, stream>>>(p);
}

}  // namespace
}  // namespace tf

extern "C" int tf_rotary_positions_fwd(const tf_rotary_io* io, void* stream) {
  using namespace tf;
  if (!io) return TF_ERR_ARG;
  const int dtype = io->dtype, batch = io->batch, seqlen = io->seqlen, q_heads = io->q_heads, k_heads = io->k_heads,
            head_dim = io->head_dim, rotary_dim = io->rotary_dim;
  const bool interleaved = io->interleaved != 0;
  const void *q = io->q, *k = io->k;
  void *q_out = io->q_out, *k_out = io->k_out;
  const int64_t* strides = io->strides;
  if (dtype != TF_F32 && dtype != TF_BF16) return TF_ERR_ARG;
  if (batch < 0 || seqlen < 0 || q_heads < 0 || k_heads < 0 || head_dim < 1 || rotary_dim < 2 || rotary_dim % 2 ||
      rotary_dim > head_dim)
    return TF_ERR_ARG;
  if (batch == 0 || seqlen == 0 || q_heads + k_heads == 0) return TF_OK;
  if (!io->positions || !io->inv_freq || (q_heads && (!q || !q_out)) || (k_heads && (!k || !k_out))) return TF_ERR_ARG;
  if (rotary_dim / 2 > kMaxPairs || static_cast<int64_t>(head_dim) * (q_heads + k_heads) > 65535) return TF_ERR_SIZE;
  RotaryParams p{};
  p.q = q, p.k = k, p.qo = q_out, p.ko = k_out;
  for (int i = 0; i < 3; ++i) {
    p.sq[i] = strides[i], p.sk[i] = strides[3 + i], p.soq[i] = strides[6 + i], p.sok[i] = strides[9 + i];
  }
  p.positions = io->positions;
  p.sp[0] = strides[12], p.sp[1] = strides[13];
  p.inv_freq = io->inv_freq;
  p.amplitude = static_cast<float>(io->amplitude);
  p.T = seqlen;
  p.tokens = static_cast<int64_t>(batch) * seqlen;
  if (p.tokens > 0x7fffffffll) return TF_ERR_SIZE;
  p.half = rotary_dim / 2;
  p.qheads = q_heads;
  // The widest vector that divides the rotated span and the rest, the strides and the addresses.
  const int size = dtype == TF_F32 ? 4 : 2;
  int vec = 16 / size;
  const int span = interleaved ? rotary_dim : p.half;
  auto fits = [&](int v) {
    if (span % v || (head_dim - rotary_dim) % v || (2 * p.half) % v) return false;
    const void* ptr[4] = {q, k, q_out, k_out};
    for (int i = 0; i < 4; ++i) {
      if (!(i % 2 ? k_heads : q_heads)) continue;
      if (reinterpret_cast<uintptr_t>(ptr[i]) % (v * size)) return false;
      const int64_t extent[3] = {batch, seqlen, i % 2 ? k_heads : q_heads};
      for (int j = 0; j < 3; ++j)
        if (extent[j] > 1 && strides[3 * i + j] % v) return false;
    }
    return true;
  };
  while (vec > 1 && !fits(vec)) vec /= 2;
  p.rot_items = interleaved && vec > 1 ? rotary_dim / vec : p.half / vec;
  const int items = p.rot_items + (head_dim - rotary_dim) / vec;
  p.items = fast_div(items);
  p.heads = fast_div(q_heads + k_heads);
  const int per_token = items * (q_heads + k_heads);
  // Several tokens a block where a token has little work, while the blocks still fill the device
  // and the index of an item stays below 2^16.
  int tile = 1;
  while (tile < kMaxTile && tile * 2 * per_token <= 2048 && tile * 2 * p.half <= kMaxPairs && p.tokens / (tile * 2) >= 4 * sm_count())
    tile *= 2;
  p.tile = tile;
  const int st = check_device();
  if (st != TF_OK) return st;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == TF_F32) {
    if (vec == 4) launch<float, 4>(p, interleaved, s);
    else if (vec == 2) launch<float, 2>(p, interleaved, s);
    else launch<float, 1>(p, interleaved, s);
  } else {
    if (vec == 8) launch<bf16, 8>(p, interleaved, s);
    else if (vec == 4) launch<bf16, 4>(p, interleaved, s);
    else if (vec == 2) launch<bf16, 2>(p, interleaved, s);
    else launch<bf16, 1>(p, interleaved, s);
  }
  return launch_status();
}
