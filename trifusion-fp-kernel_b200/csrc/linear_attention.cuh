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

}  // namespace tf
