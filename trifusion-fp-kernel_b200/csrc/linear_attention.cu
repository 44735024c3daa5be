// Linear attention with a decay for each head, and a carried state:
//
//   S_t = e^{g_t} S_{t-1} + k_t v_t^T      (N x P, FP32)
//   o_t = scale * q_t S_t
//
// q and k heads are shared by H / Hq heads of v. This file holds the recurrent
// form (one token after another, the state in registers); linear_chunks.cu the
// chunked form on the tensor cores.
#include <type_traits>

#include "../../include/trifusion_b200.h"
#include "linear_attention.cuh"
#include "tf_common.cuh"
#include "tf_host.cuh"

namespace tf {
namespace {

__device__ __forceinline__ float ld_f(const float* p) { return __ldg(p); }
__device__ __forceinline__ float ld_f(const bf16* p) { return bf2f(__ldg(p)); }
__device__ __forceinline__ void st_f(float* p, float x) { *p = x; }
__device__ __forceinline__ void st_f(bf16* p, float x) { *p = __float2bfloat16_rn(x); }

// The factor e^g of a log decay g. Rounded to FP32, errors of the factor add up over a long memory
// (3e-9 a token, all one way: 1.7e-5 of the state after 4680 tokens of slow decay, now 1.1e-6). So
// near 1 it is e^g rounded down, and what that leaves is applied too: with the factor of a next token,
// or as a second factor. Both are above zero for every finite g, so that an infinite state stays
// what it is (S + (e^g - 1) S would be inf - inf). 0 gives exactly 1, -inf exactly 0, NaN stays.
constexpr float kTiny = 0x1p-149f;  // FP32's smallest number
__device__ __forceinline__ bool near_one(float g) { return g <= 0.f && g > -0.35f; }
// e^g - 1 by its Taylor series to g^7: the rest is below 2^-25 of it where near_one(g).
__device__ __forceinline__ float decay_less_one(float g) {
  float x = 1.f / 5040.f;
  x = fmaf(x, g, 1.f / 720.f);
  x = fmaf(x, g, 1.f / 120.f);
  x = fmaf(x, g, 1.f / 24.f);
  x = fmaf(x, g, 1.f / 6.f);
  x = fmaf(x, g, 0.5f);
  return fmaf(x, g * g, g);
}
// 1 + x for -0.35 < x < 2^-24, rounded down; x is left with the rest (both differences are exact).
__device__ __forceinline__ float take_factor(float& x) {
  const float down = __fadd_rd(1.f, x);
  x = (1.f - down) + x;
  return down;
}
__device__ __forceinline__ float far_factor(float g) {
  const float e = ex2_approx(g * kLog2e);
  return e == 0.f && g > -INFINITY ? kTiny : e;
}

// ---- recurrent form ------------------------------------------------------------
// One block: one row, one head, 32 columns of its state. Thread (warp w, lane l) holds columns
// 4 (l % 8) .. +3 of the NR rows from (4 w + l / 8) NR on: a token's q, k and v are wide reads of
// shared memory, its output three shuffles (each halves what a lane still sums) and a partial sum
// of each warp. Tokens come in batches: while one is worked on, the next one's operands are in shared
// memory and those of the one after it on their way to registers, and a batch takes one barrier,
// behind which every warp sums up the output of some of its tokens. Bound by issue and, with few
// blocks, by the latency of a token's chain. Up to two blocks an SM, eight warps with a whole batch
// unrolled are faster, else four warps with half of it (fewer instructions for a token). FP32, us:
//   1 x 7 tokens, 12 heads, N 128, P 64        24 blocks     eight 4.5   four  4.9
//   2 x 3600, 12 heads, N 128, P 64            48 blocks     eight 590   four  758
//   12 x 200, 12 heads, N 128, P 64           288 blocks     eight 52.1  four 61.0
//   16 x 200, 12 heads, N 128, P 64           384 blocks     eight 83.0  four 78.4
//   8 x 4097, 32 heads, N 64, P 64            512 blocks     eight 1494  four 1190
//   32 x 7, 32 heads, N 128, P 64            2048 blocks     eight 33.0  four 24.1
// (2 x 3600, each against the kernel of its time: a barrier for every token 1058 against 510 us; a
// column a lane 800 against 510; the next batch loaded while one is worked on, not two, 694 against
// 604; both parts of a factor applied to each token 625 against 607.)
template <typename T, int NR, int WARPS>
__global__ void __launch_bounds__(32 * WARPS, NR == 8 ? 4 : 2) linear_scan_kernel(const __grid_constant__ LinearParams p) {
  constexpr int kThreads = 32 * WARPS, kRows = 4 * WARPS * NR;
  constexpr int kBatch = kRows > 128 ? 4 : 8;  // tokens
  constexpr int kOwn = kBatch / WARPS;         // of them a warp brings the v, and sums up the output
  constexpr int kLoads = kBatch * kRows / kThreads;  // of q, and of k, by a thread
  constexpr int kUnroll = WARPS == 8 ? kBatch : 4;
  static_assert(kBatch % WARPS == 0 && kBatch * kRows % kThreads == 0, "a batch is shared out evenly");
  __shared__ alignas(16) float kq[2][kBatch][2][kRows];
  __shared__ alignas(16) float vs[2][kBatch][32];
  __shared__ float as[2][kBatch], rest, partial[2][kBatch][WARPS][32];
  const int slices = (p.P + 31) / 32;
  const int slice = blockIdx.x % slices;
  const int row = blockIdx.x / slices;
  const int h = row % p.H, b = row / p.H;
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r0 = (4 * w + (lane >> 3)) * NR, c0 = slice * 32 + 4 * (lane & 7);  // of the state
  const int col = slice * 32 + lane;  // of v and the output
  const bool on = col < p.P;

  const int64_t slot = p.slots ? p.slots[b] : b;
  const bool in_pool = p.state && slot >= 0 && slot < p.nslots;
  float* st = p.state + (in_pool ? slot * p.ss[0] + h * p.ss[1] + static_cast<int64_t>(r0) * p.P + c0 : 0);
  float2 s[4][NR / 2];  // [column][pair of rows]
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const float4 x = in_pool && !p.fresh && c0 < p.P && r0 + i < p.N ? *reinterpret_cast<const float4*>(st + i * p.P)
                                                                     : make_float4(0.f, 0.f, 0.f, 0.f);
    (i % 2 ? s[0][i / 2].y : s[0][i / 2].x) = x.x;
    (i % 2 ? s[1][i / 2].y : s[1][i / 2].x) = x.y;
    (i % 2 ? s[2][i / 2].y : s[2][i / 2].x) = x.z;
    (i % 2 ? s[3][i / 2].y : s[3][i / 2].x) = x.w;
  }
  bool taken = false;  // an earlier row has this slot
  if (p.slots) {
    if (in_pool)
      for (int i = threadIdx.x; i < b; i += kThreads) taken |= p.slots[i] == slot;
    taken = __syncthreads_or(taken);
  }
  int64_t len = p.T;
  if (p.lengths) len = min(max(p.lengths[b], static_cast<int64_t>(0)), len);
  T* out = static_cast<T*>(p.out) + b * p.so[0] + h * p.so[2] + col;
  if (p.state && (!in_pool || taken)) {
    // No state of its own: zeros for a row that is padding, NaN for one that names a wrong slot.
    const float fill = slot < 0 ? 0.f : __int_as_float(0x7fc00000);
    if (on)
      for (int64_t t = w; t < p.T; t += WARPS) st_f(out + t * p.so[1], t < len ? fill : 0.f);
    return;
  }
  const int hq = h / (p.H / p.Hq);
  const T* q = static_cast<const T*>(p.q) + b * p.sq[0] + hq * p.sq[2];
  const T* k = static_cast<const T*>(p.k) + b * p.sk[0] + hq * p.sk[2];
  const T* v = static_cast<const T*>(p.v) + b * p.sv[0] + h * p.sv[2] + col;
  const float* g = p.decay + b * p.sg[0] + h * p.sg[1];
  // What a thread brings of the batch from t0 on. Tokens past the length change nothing: zeros, and
  // no decay.
  float kn[kLoads], qn[kLoads], vn[kOwn], gn, left = 0.f;
  auto load = [&](int64_t t0) {
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int i = threadIdx.x + j * kThreads, n = i % kRows;
      const int64_t t = t0 + i / kRows;
      const bool live = t < len && n < p.N;
      kn[j] = live ? ld_f(k + t * p.sk[1] + n) : 0.f;
      qn[j] = live ? ld_f(q + t * p.sq[1] + n) : 0.f;
    }
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
      const int64_t t = t0 + w * kOwn + j;
      vn[j] = t < len && on ? ld_f(v + t * p.sv[1]) : 0.f;
    }
    gn = threadIdx.x < kBatch && t0 + threadIdx.x < len ? g[(t0 + threadIdx.x) * p.sg[2]] : 0.f;
  };
  auto store = [&](int x) {
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int i = threadIdx.x + j * kThreads;
      kq[x][i / kRows][0][i % kRows] = kn[j], kq[x][i / kRows][1][i % kRows] = qn[j];
    }
#pragma unroll
    for (int j = 0; j < kOwn; ++j) vs[x][w * kOwn + j][lane] = vn[j];
    if (w == 0) {  // token after token, each with what the factors before it left
      const float own = near_one(gn) ? decay_less_one(gn) : 0.f;
      float factor = far_factor(gn);
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        left += __shfl_sync(0xffffffffu, own, j);
        const float near = take_factor(left);
        if (lane == j && near_one(gn)) factor = near;
      }
      if (lane < kBatch) as[x][lane] = factor;
      if (lane == 0) rest = left;
    }
  };
  bool resetting = false;
#pragma unroll 1
  for (int64_t t = threadIdx.x; t < len; t += kThreads) resetting |= g[t * p.sg[2]] == -INFINITY;
  load(0);
  store(0);
  load(kBatch);
  resetting = __syncthreads_or(resetting);
  auto batches = [&](auto resets) {
    int x = 0;
    for (int64_t t0 = 0; t0 < len; t0 += kBatch, x ^= 1) {
      store(x ^ 1);
      load(t0 + 2 * kBatch);
#pragma unroll (decltype(resets)::value ? 1 : kUnroll)
      for (int t = 0; t < kBatch; ++t) {
        const float a = as[x][t];
        const float2 factor = make_float2(a, a);
        if (decltype(resets)::value && a == 0.f) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int i = 0; i < NR / 2; ++i) s[c][i] = make_float2(0.f, 0.f);
        }
        const float4 vr = *reinterpret_cast<const float4*>(&vs[x][t][4 * (lane & 7)]);
        const float2 vv[4] = {make_float2(vr.x, vr.x), make_float2(vr.y, vr.y), make_float2(vr.z, vr.z),
                              make_float2(vr.w, vr.w)};
        float2 o[4] = {};
#pragma unroll
        for (int i = 0; i < NR / 2; ++i) {
          const float2 kk = *reinterpret_cast<const float2*>(&kq[x][t][0][r0 + 2 * i]);
          const float2 qq = *reinterpret_cast<const float2*>(&kq[x][t][1][r0 + 2 * i]);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            s[c][i] = fma2(factor, s[c][i], mul2(kk, vv[c]));
            o[c] = fma2(qq, s[c][i], o[c]);
          }
        }
        const bool hi = lane & 8, top = lane & 16;
        float y[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) y[c] = o[c].x + o[c].y;
        float y0 = hi ? y[2] : y[0], y1 = hi ? y[3] : y[1];
        y0 += __shfl_xor_sync(0xffffffffu, hi ? y[0] : y[2], 8);
        y1 += __shfl_xor_sync(0xffffffffu, hi ? y[1] : y[3], 8);
        const float z = __shfl_xor_sync(0xffffffffu, top ? y0 : y1, 16) + (top ? y1 : y0);
        partial[x][t][w][4 * (lane & 7) + (hi ? 2 : 0) + (top ? 1 : 0)] = z;
      }
      __syncthreads();
      if (on) {
#pragma unroll
        for (int j = 0; j < kOwn; ++j) {
          const int t = w * kOwn + j;
          float sum = 0.f;
#pragma unroll
          for (int i = 0; i < WARPS; ++i) sum += partial[x][t][i][lane];
          if (t0 + t < len) st_f(out + (t0 + t) * p.so[1], sum * p.scale);
        }
      }
    }
  };
  // A decay of -inf forgets what is not finite too, which a product would not. Rows with one have a loop
  // of their own: its branch for every token keeps tokens from overlapping (FP32, 2 x 3600: 643 us).
  if (resetting) batches(std::true_type());
  else batches(std::false_type());
  if (on)
    for (int64_t t = len + w; t < p.T; t += WARPS) st_f(out + t * p.so[1], 0.f);
  if (p.state && c0 < p.P && (len > 0 || p.fresh)) {
    const float more = fmaxf(rest, kTiny);  // what the factors left
#pragma unroll
    for (int i = 0; i < NR; ++i)
      if (r0 + i < p.N) {
        auto at = [&](int c) {
          const float y = i % 2 ? s[c][i / 2].y : s[c][i / 2].x;
          return fmaf(more, y, y);
        };
        *reinterpret_cast<float4*>(st + i * p.P) = make_float4(at(0), at(1), at(2), at(3));
      }
  }
}

constexpr int kStepThreads = 256;

// One token. Thread (warp w, lane l) holds columns 4 (l % 8) .. +3 of state rows w * 4 + l / 8 +
// 32 i, on up to CS times 32 columns, so that a warp reads four 128-byte row segments at a time, a
// block has 16 KB of state on its way where N <= 128, and the sum over rows for the output is two
// shuffles and eight partial sums in shared memory. Bound by HBM: the states are
// read and written once. They are streamed (evict-first): larger pools than the L2 would only
// push each other out, smaller ones stay in it all the same. 64 rows of 32 heads, 128 x 128:
// 43.5 us (268 MB, 94 % of the measured copy rate); 48.0 us with ordinary accesses, 45.1 and
// 46.6 us with four and six blocks an SM instead of five.
template <typename T, int NR, int CS>
__global__ void __launch_bounds__(kStepThreads, NR > 4 ? 3 : NR == 4 ? 5 : CS == 1 ? 6 : 4)
    linear_step_kernel(const __grid_constant__ LinearParams p) {
  __shared__ float4 partial[CS][8][8];
  const int slices = (p.P + 32 * CS - 1) / (32 * CS);
  const int slice = blockIdx.x % slices;
  const int row = blockIdx.x / slices;
  const int h = row % p.H, b = row / p.H;
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int col = slice * 32 * CS + 4 * (lane & 7);  // and 32 columns on, CS - 1 times
  const int r0 = w * 4 + (lane >> 3);
  const int64_t slot = p.slots ? p.slots[b] : b;
  const bool in_pool = slot >= 0 && slot < p.nslots;
  float* st = p.state + (in_pool ? slot * p.ss[0] + h * p.ss[1] + static_cast<int64_t>(r0) * p.P + col : 0);
  float4 s[CS][NR];
#pragma unroll
  for (int c = 0; c < CS; ++c)
#pragma unroll
    for (int i = 0; i < NR; ++i)
      if (in_pool && col + 32 * c < p.P && r0 + 32 * i < p.N)
        s[c][i] = __ldcs(reinterpret_cast<const float4*>(st + 32 * i * p.P + 32 * c));
  const int hq = h / (p.H / p.Hq);
  const T* q = static_cast<const T*>(p.q) + b * p.sq[0] + hq * p.sq[2] + r0;
  const T* k = static_cast<const T*>(p.k) + b * p.sk[0] + hq * p.sk[2] + r0;
  const T* v = static_cast<const T*>(p.v) + b * p.sv[0] + h * p.sv[2] + col;
  constexpr bool kEarly = NR <= 2;  // k and q on their way with the state, as registers allow
  float early[2][kEarly ? NR : 1] = {}, vv[CS][4] = {};
  if (kEarly) {
#pragma unroll
    for (int i = 0; i < NR; ++i)
      if (r0 + 32 * i < p.N) early[0][i % (kEarly ? NR : 1)] = ld_f(k + 32 * i), early[1][i % (kEarly ? NR : 1)] = ld_f(q + 32 * i);
  }
#pragma unroll
  for (int c = 0; c < CS; ++c)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (col + 32 * c < p.P) vv[c][j] = ld_f(v + 32 * c + j);
  const float g = p.decay[b * p.sg[0] + h * p.sg[1]];
  float more = near_one(g) ? decay_less_one(g) : 0.f, a = take_factor(more);
  if (!near_one(g)) a = far_factor(g);
  bool dead = !in_pool;  // no state of its own
  if (p.slots) {
    for (int i = threadIdx.x; i < b; i += kStepThreads) dead |= p.slots[i] == slot;
    dead = __syncthreads_or(dead);
  }
  if (a == 0.f) {  // -inf forgets what is not finite too, which a product would not
#pragma unroll
    for (int c = 0; c < CS; ++c)
#pragma unroll
      for (int i = 0; i < NR; ++i) s[c][i] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  const float2 a0 = make_float2(a, a), a1 = make_float2(fmaxf(more, kTiny), fmaxf(more, kTiny));
  float4 o[CS];
#pragma unroll
  for (int c = 0; c < CS; ++c) o[c] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    if (!dead && (CS > 1 || col < p.P) && r0 + 32 * i < p.N) {
      const float kn = kEarly ? early[0][i % (kEarly ? NR : 1)] : ld_f(k + 32 * i);
      const float qn = kEarly ? early[1][i % (kEarly ? NR : 1)] : ld_f(q + 32 * i);
#pragma unroll
      for (int c = 0; c < CS; ++c)
        if (CS == 1 || col + 32 * c < p.P) {
          float4& x = s[c][i];
          const float2 k2 = make_float2(kn, kn), q2 = make_float2(qn, qn);
          const float2 lo = make_float2(x.x, x.y), hi = make_float2(x.z, x.w);
          const float2 y = fma2(a0, lo, fma2(a1, lo, mul2(k2, make_float2(vv[c][0], vv[c][1]))));
          const float2 z = fma2(a0, hi, fma2(a1, hi, mul2(k2, make_float2(vv[c][2], vv[c][3]))));
          x = make_float4(y.x, y.y, z.x, z.y);
          const float2 oy = fma2(q2, y, make_float2(o[c].x, o[c].y)), oz = fma2(q2, z, make_float2(o[c].z, o[c].w));
          o[c] = make_float4(oy.x, oy.y, oz.x, oz.y);
          __stcs(reinterpret_cast<float4*>(st + 32 * i * p.P + 32 * c), x);
        }
    }
  }
#pragma unroll
  for (int c = 0; c < CS; ++c) {
#pragma unroll
    for (int d = 8; d < 32; d <<= 1) {
      o[c].x += __shfl_xor_sync(0xffffffffu, o[c].x, d);
      o[c].y += __shfl_xor_sync(0xffffffffu, o[c].y, d);
      o[c].z += __shfl_xor_sync(0xffffffffu, o[c].z, d);
      o[c].w += __shfl_xor_sync(0xffffffffu, o[c].w, d);
    }
    if (lane < 8) partial[c][w][lane] = o[c];
  }
  __syncthreads();
  const int c = (slice * CS + w) * 32 + lane;
  if (w < CS && c < p.P) {
    const float* f = reinterpret_cast<const float*>(&partial[w][0][0]);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += f[32 * i + lane];
    // A row without a state: zero where it is padding, NaN where it names a wrong slot.
    const float y = dead ? (slot < 0 ? 0.f : __int_as_float(0x7fc00000)) : sum * p.scale;
    st_f(static_cast<T*>(p.out) + b * p.so[0] + h * p.so[2] + c, y);
  }
}

template <typename T, int NR>  // N <= 32 NR
void launch_rows(const LinearParams& p, cudaStream_t stream) {
  const int64_t rows = static_cast<int64_t>(p.B) * p.H;
  if (p.T == 1 && p.state && !p.fresh && !p.lengths) {
    // As many columns a block as make up 16 KB, and as there are.
    auto step = [&](auto cs) {
      constexpr int CS = decltype(cs)::value;
      linear_step_kernel<T, NR, CS>
          <<<static_cast<unsigned>(rows * ((p.P + 32 * CS - 1) / (32 * CS))), kStepThreads, 0, stream>>>(p);
    };
    if (NR == 1 && p.P > 64) step(std::integral_constant<int, NR == 1 ? 4 : 1>());
    else if (NR <= 2 && p.P > 32) step(std::integral_constant<int, NR <= 2 ? 2 : 1>());
    else step(std::integral_constant<int, 1>());
  } else {
    auto scan = [&](auto warps) {
      constexpr int W = decltype(warps)::value, R = 8 * NR / W < 2 ? 2 : 8 * NR / W;
      linear_scan_kernel<T, R, W><<<static_cast<unsigned>(rows * ((p.P + 31) / 32)), 32 * W, 0, stream>>>(p);
    };
    if (NR <= 4 && rows * ((p.P + 31) / 32) <= 2 * sm_count()) scan(std::integral_constant<int, NR <= 4 ? 8 : 4>());
    else scan(std::integral_constant<int, 4>());
  }
}
template <typename T>
void launch_scan(const LinearParams& p, cudaStream_t stream) {
  if (p.N <= 32) launch_rows<T, 1>(p, stream);
  else if (p.N <= 64) launch_rows<T, 2>(p, stream);
  else if (p.N <= 128) launch_rows<T, 4>(p, stream);
  else launch_rows<T, 8>(p, stream);
}

}  // namespace
}  // namespace tf

extern "C" {

int tf_linear_attention_chunked(int batch, int seqlen, int heads, int groups, int key_dim, int value_dim, int dtype) {
  if (batch <= 0 || seqlen <= 0 || heads <= 0 || groups <= 0 || heads % groups || key_dim <= 0 || value_dim <= 0)
    return 0;
  return tf::linear_chunk_workspace(batch, seqlen, heads, groups, key_dim, value_dim, dtype) >= 0;
}

int64_t tf_linear_attention_workspace_size(int batch, int seqlen, int heads, int groups, int key_dim, int value_dim,
                                           int dtype) {
  if (!tf_linear_attention_chunked(batch, seqlen, heads, groups, key_dim, value_dim, dtype)) return 0;
  return tf::linear_chunk_workspace(batch, seqlen, heads, groups, key_dim, value_dim, dtype);
}

int tf_linear_attention_fwd(const tf_linear_attention_io* io, void* stream) {
  using namespace tf;
  if (!io) return TF_ERR_ARG;
  const int dtype = io->dtype, batch = io->batch, seqlen = io->seqlen, heads = io->heads, groups = io->groups,
            key_dim = io->key_dim, value_dim = io->value_dim;
  const int64_t state_slots = io->state_slots;
  float* state = io->state;
  if (dtype != TF_F32 && dtype != TF_BF16) return TF_ERR_ARG;
  if (batch < 0 || seqlen < 0 || heads < 0 || groups < 1 || heads % groups || state_slots < 0) return TF_ERR_ARG;
  if (key_dim < 8 || value_dim < 8 || key_dim % 8 || value_dim % 8 || key_dim > 256 || value_dim > 256)
    return TF_ERR_ARG;
  if (io->slots && !state) return TF_ERR_ARG;
  if (!io->slots && state && state_slots < batch) return TF_ERR_ARG;
  if (batch == 0 || heads == 0 || (seqlen == 0 && !(state && io->fresh))) return TF_OK;
  if (seqlen > 0 && (!io->q || !io->k || !io->v || !io->decay || !io->out)) return TF_ERR_ARG;
  LinearParams p{};
  p.q = io->q, p.k = io->k, p.v = io->v, p.out = io->out;
  p.decay = io->decay;
  p.state = state;
  p.nslots = state_slots;
  p.fresh = io->fresh != 0;
  p.slots = io->slots;
  p.lengths = io->lengths;
  const int64_t* s = io->strides;
  for (int i = 0; i < 3; ++i) p.sq[i] = s[i], p.sk[i] = s[3 + i], p.sv[i] = s[6 + i], p.sg[i] = s[9 + i], p.so[i] = s[12 + i];
  p.ss[0] = s[15], p.ss[1] = s[16];
  if (state && (reinterpret_cast<uintptr_t>(state) % 16 || (state_slots > 1 && p.ss[0] % 4) || (heads > 1 && p.ss[1] % 4)))
    return TF_ERR_LAYOUT;
  p.B = batch, p.T = seqlen, p.H = heads, p.Hq = groups, p.N = key_dim, p.P = value_dim;
  p.scale = static_cast<float>(io->scale);
  if (static_cast<int64_t>(batch) * heads * ((value_dim + 31) / 32) > 0x7fffffffll || seqlen > 0x7fffff00)
    return TF_ERR_SIZE;
  int st = check_device();
  if (st != TF_OK) return st;
  if (linear_chunk_workspace(batch, seqlen, heads, groups, key_dim, value_dim, dtype) >= 0) {
    st = launch_linear_chunks(p, dtype, io->workspace, io->workspace_bytes, static_cast<cudaStream_t>(stream));
    if (st >= 0) return st;
  }
  if (dtype == TF_F32) launch_scan<float>(p, static_cast<cudaStream_t>(stream));
  else launch_scan<bf16>(p, static_cast<cudaStream_t>(stream));
  return launch_status();
}

}  // extern "C"
