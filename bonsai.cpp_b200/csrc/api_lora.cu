// C ABI of the adapter sets (include/bonsai_cuda.h).
#include "../../include/bonsai_cuda.h"
#include "internal.cuh"

#include <cmath>

using namespace bonsai;

extern "C" {

int bonsai_lora_create(int out_dim, int in_dim, int max_rank, int n_slots, int swiglu_from, bonsai_lora_t* out) {
  if (!out) return fail(BONSAI_ERR_ARG, "lora_create: null output handle");
  *out = nullptr;
  if (out_dim <= 0 || in_dim <= 0 || n_slots <= 0) return fail(BONSAI_ERR_ARG, "lora_create: non-positive shape");
  if (in_dim % BONSAI_B1_BLOCK_SIZE != 0) return fail(BONSAI_ERR_ARG, "lora_create: in_dim must be a multiple of 32");
  if (max_rank < 1 || max_rank > 128) return fail(BONSAI_ERR_UNSUPPORTED, "lora_create: max_rank must be 1..128");
  if (swiglu_from >= 0 && (swiglu_from >= out_dim || ((out_dim - swiglu_from) & 1) || (swiglu_from & 1)))
    return fail(BONSAI_ERR_ARG, "lora_create: swiglu_from must be even and leave an even number of rows");
  auto* h = new bonsai_lora();
  LoraDevice& s = h->set;
  s.n_rows = out_dim;
  s.k_in = in_dim;
  s.max_rank = max_rank;
  s.r_pad = (max_rank + 15) / 16 * 16;
  s.n_slots = n_slots;
  s.n_ftiles = (out_dim + 127) / 128;
  s.swiglu_from = swiglu_from < 0 ? -1 : swiglu_from;
  cudaGetDevice(&s.device);
  const size_t down = (size_t)n_slots * s.r_pad * in_dim * sizeof(__half);
  const size_t up = (size_t)n_slots * s.r_pad * s.n_ftiles * 128 * sizeof(__half);
  if (cudaMalloc(reinterpret_cast<void**>(&s.down), down) != cudaSuccess ||
      cudaMalloc(reinterpret_cast<void**>(&s.up), up) != cudaSuccess ||
      cudaMalloc(reinterpret_cast<void**>(&s.info), n_slots * sizeof(LoraSlot)) != cudaSuccess) {
    cudaGetLastError();
    bonsai_lora_free(h);
    return fail(BONSAI_ERR_NOMEM, "lora_create: device allocation failed");
  }
  cudaError_t e = cudaMemset(s.info, 0, n_slots * sizeof(LoraSlot));  // rank 0: every slot empty
  if (e == cudaSuccess) e = cudaDeviceSynchronize();
  if (e != cudaSuccess) {
    bonsai_lora_free(h);
    return cuda_status(e, "lora_create: clear");
  }
  *out = h;
  return 0;
}

int bonsai_lora_set(bonsai_lora_t h, int slot, const uint16_t* down, const uint16_t* up, int rank, float scale,
                    void* stream) {
  if (!h) return fail(BONSAI_ERR_ARG, "lora_set: null handle");
  const LoraDevice& s = h->set;
  if (slot < 0 || slot >= s.n_slots) return fail(BONSAI_ERR_ARG, "lora_set: no such slot");
  if (rank < 0 || rank > s.max_rank) return fail(BONSAI_ERR_ARG, "lora_set: rank outside [0, max_rank]");
  if (rank > 0 && (!down || !up)) return fail(BONSAI_ERR_ARG, "lora_set: null adapter");
  if (rank > 0 && !std::isfinite(scale)) return fail(BONSAI_ERR_ARG, "lora_set: scale must be finite");
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_status(e, "lora_set: cudaGetDevice");
  if (dev != s.device) return fail(BONSAI_ERR_ARG, "lora_set: the adapters live on device " + std::to_string(s.device));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const LoraSlot info{rank, scale};
  if (rank == 0) return launch_lora_retile(nullptr, info, s, slot, st);
  __half* d = s.down + (size_t)slot * s.r_pad * s.k_in;
  const size_t row = (size_t)s.k_in * sizeof(__half), u_bytes = (size_t)rank * s.n_rows * sizeof(__half);
  e = cudaMemcpyAsync(d, down, rank * row, cudaMemcpyDefault, st);
  if (e == cudaSuccess && rank < s.r_pad)
    e = cudaMemsetAsync(d + (size_t)rank * s.k_in, 0, (s.r_pad - rank) * row, st);
  if (e != cudaSuccess) return cuda_status(e, "lora_set: copy");
  cudaPointerAttributes at{};
  if (cudaPointerGetAttributes(&at, up) == cudaSuccess && at.type == cudaMemoryTypeDevice && at.device == dev)
    return launch_lora_retile(reinterpret_cast<const __half*>(up), info, s, slot, st);
  cudaGetLastError();
  void* staged = nullptr;
  int rc = scratch_alloc(&staged, u_bytes, "lora_set", st);
  if (rc) return rc;
  e = cudaMemcpyAsync(staged, up, u_bytes, cudaMemcpyDefault, st);
  rc = e == cudaSuccess ? launch_lora_retile(static_cast<const __half*>(staged), info, s, slot, st)
                        : cuda_status(e, "lora_set: copy");
  scratch_free(staged, st);
  return rc;
}

int bonsai_lora_free(bonsai_lora_t h) {
  if (!h) return 0;
  cudaFree(h->set.down);
  cudaFree(h->set.up);
  cudaFree(h->set.info);
  delete h;
  return 0;
}

}  // extern "C"
