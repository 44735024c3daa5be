// Parameters of the linear-attention launches (linear_attention.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace tf {

struct LinearParams {
  const void *q, *k, *v;
  void* out;
  const float* decay;       // [B, H, T] natural log
  float* state;             // [slots, H, N, P], or NULL
  int64_t nslots;
  const int64_t* slots;     // [B], or NULL: row b has slot b
  const int64_t* lengths;   // [B], or NULL
  int64_t sq[3], sk[3], sv[3], so[3];  // batch, time, head (elements)
  int64_t sg[3];                       // batch, head, time
  int64_t ss[2];                       // slot, head
  int B, T, H, Hq, N, P;
  int fresh;                // the state is written but not read: it starts at zero
  float scale;
};

// The chunked form (linear_chunks.cu): bytes of workspace it takes, -1 where it does not
// apply; a launch of it, or -1 where a tensor's layout does not allow it.
int64_t linear_chunk_workspace(int B, int T, int H, int Hq, int N, int P, int dtype);
int launch_linear_chunks(const LinearParams& l, int dtype, void* workspace, int64_t workspace_bytes,
                         cudaStream_t stream);
int read_linear_error(int reset);
int* host_error_word();
unsigned long long flag_wait_limit_ns();

// Two FP32 products, or products and sums, in one instruction.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mul.rn.f32x2 z, x, y;\n"
      " mov.b64 {%0, %1}, z;\n}\n"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n .reg .b64 x, y, z, w;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mov.b64 w, {%6, %7};\n"
      " fma.rn.f32x2 z, x, y, w;\n mov.b64 {%0, %1}, z;\n}\n"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}

}  // namespace tf
