// common.cuh — shared declarations of the libenigma_cuda translation units.
#pragma once
#include <cstdint>
#include <cuda_runtime.h>
#include <cuda_bf16.h>

#include "../../include/enigma_cuda.h"
#include "sm100.cuh"

namespace enigma {

// SM count of the current device (cached per device).
int sm_count();

// Device word that bounded waits set on timeout (one per device, zeroed at init; created
// by the first call, nullptr if that allocation fails).
uint32_t* device_status();
// The same word if it already exists on the current device, else nullptr (never allocates).
uint32_t* device_status_if_exists();
// A pair of work counters of the current device for one launch (a dynamic work queue:
// [0] next item, [1] spare), taken round-robin from a per-device pool so launches in flight
// on different streams use different pairs; the caller zeroes it on its stream before the
// launch.  nullptr if the per-device state could not be created.
uint32_t* work_counters();
// Reads and clears the no-allocation decode entry's status word on the current device
// (0 if that entry has not run there).  Allocates nothing.
cudaError_t noalloc_take_status(uint32_t* value);
// One CTA that waits on a barrier nothing arrives on, gives up after `polls` polls and
// flags *status as a timed-out bounded wait does.
cudaError_t launch_timeout_probe(uint32_t* status, long long polls, cudaStream_t s);

// Operator launchers (asynchronous).  Arguments are validated by the C ABI layer.
cudaStream_t aux_stream();
cudaError_t rmsnorm_launch(int dtype, const void* x, const void* w, void* y, int64_t rows,
                           int64_t hidden, float eps, cudaStream_t s);
// Same, with the SM count given (no per-device state is touched).
cudaError_t rmsnorm_launch_sms(int dtype, const void* x, const void* w, void* y, int64_t rows,
                               int64_t hidden, float eps, int sms, cudaStream_t s);
// The decode step's input norm (bf16): launched as a programmatic dependent when the row
// is at most 128 16-byte vectors (hidden <= 1024), so in a layer stack it is resident
// before the previous layer's last kernel ends; else the same as rmsnorm_launch_sms.
cudaError_t rmsnorm_launch_pdl_bf16(const void* x, const void* w, void* y, int64_t rows,
                                    int64_t hidden, float eps, int sms, cudaStream_t s);
cudaError_t gemm_bf16_launch(const void* A, const void* B, void* C, int64_t M, int64_t N,
                             int64_t K, cudaStream_t s);
cudaError_t gemm_f32_launch(const void* A, const void* B, void* C, int64_t M, int64_t N,
                            int64_t K, bool accumulate, cudaStream_t s);
cudaError_t gemm_f32_trans_launch(const void* A, const void* B, void* C, int64_t M, int64_t N,
                                  int64_t K, bool trans_a, bool trans_b, bool accumulate,
                                  cudaStream_t s);
cudaError_t sdpa_f32_launch(const void* Q, const void* K, const void* V, void* O, int64_t B,
                            int64_t Hq, int64_t Hkv, int64_t Sq, int64_t Skv, int64_t D,
                            float scale, bool causal, cudaStream_t s);
cudaError_t sdpa_strided_launch(int dtype, const void* Q, const void* K, const void* V, void* O,
                                int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t Skv,
                                int64_t D, const int64_t* strides12, float scale, bool causal,
                                const float* sinks, cudaStream_t s);
cudaError_t sdpa_bf16_launch(const void* Q, const void* K, const void* V, void* O, int64_t B,
                             int64_t Hq, int64_t Hkv, int64_t Sq, int64_t Skv, int64_t D,
                             float scale, bool causal, cudaStream_t s);

size_t decode_workspace_bytes(const enigma_decode_layer_desc& d);
cudaError_t decode_layer_launch(const enigma_decode_layer_desc& d, const void* x, void* out,
                                void* ws, cudaStream_t s);

// Argument checks of a decode-layer descriptor (ENIGMA_OK or ENIGMA_ERR_BADARG + message).
int32_t check_decode_desc(const enigma_decode_layer_desc* d);

cudaError_t qwen_decode_f32_launch(const enigma_qwen_decode_f32_desc& q, cudaStream_t s);

// Serving attention: bf16 shapes that fit the tensor-core kernels' tiles go there, the rest to
// the CUDA-core kernels.
cudaError_t sdpa_packed_launch(const enigma_sdpa_packed_desc& d, cudaStream_t s);
cudaError_t sdpa_packed_simt_launch(const enigma_sdpa_packed_desc& d, cudaStream_t s);
// blocked: the parts' layout is [slot][D / 8][128][8], else [slot][128][D].
cudaError_t sdpa_packed_join_launch(const enigma_sdpa_packed_desc& d, bool blocked, cudaStream_t s);
size_t sdpa_shared_prefix_workspace(const enigma_sdpa_shared_prefix_desc& d);
cudaError_t sdpa_shared_prefix_launch(const enigma_sdpa_shared_prefix_desc& d, cudaStream_t s);
cudaError_t sdpa_paged_simt_launch(const enigma_sdpa_shared_prefix_desc& d, cudaStream_t s);

// Paged cache (kv_cache.cu).
size_t kv_cache_workspace_bytes(const enigma_kv_cache_desc& d);
cudaError_t kv_cache_fork(const enigma_kv_cache_desc& d, const int32_t* parents,
                          const int32_t* children, int64_t n, cudaStream_t s);
cudaError_t kv_cache_free(const enigma_kv_cache_desc& d, const int32_t* slots, int64_t n,
                          cudaStream_t s);
cudaError_t kv_cache_reserve(const enigma_kv_cache_desc& d, const int32_t* slots,
                             const int32_t* lens, int64_t n, cudaStream_t s);
cudaError_t kv_cache_write(const enigma_kv_cache_desc& d, int64_t layer, const void* new_k,
                           const void* new_v, const int64_t* strides4, const int32_t* slots,
                           const int32_t* starts, const int32_t* cu, int64_t n, int64_t tokens,
                           cudaStream_t s);
cudaError_t kv_cache_compact(const enigma_kv_cache_desc& d, cudaStream_t s);
cudaError_t kv_cache_copy_pages(const enigma_kv_cache_desc& d, const int32_t* src,
                                const int32_t* dst, int64_t n, cudaStream_t s);

// The whole pages that the last fork or compaction of this map copied, in other buffers that hold one
// page for each of its pages (at most n).
cudaError_t kv_cache_copy_listed(const enigma_kv_cache_desc& d, int64_t n, cudaStream_t s);

// Rotary positions (rope.cu).
cudaError_t rope_launch(const enigma_rope_desc& d, cudaStream_t s);

// The cache in 8-bit codes (kv_cache_codes8.cu) and attention over it (attn_codes8.cu).
cudaError_t kv_cache_q8_fork(const enigma_kv_cache_q8_desc& d, const int32_t* parents,
                             const int32_t* children, int64_t n, cudaStream_t s);
cudaError_t kv_cache_q8_compact(const enigma_kv_cache_q8_desc& d, cudaStream_t s);
cudaError_t kv_cache_q8_copy_pages(const enigma_kv_cache_q8_desc& d, const int32_t* src,
                                   const int32_t* dst, int64_t n, cudaStream_t s);
cudaError_t kv_cache_q8_write(const enigma_kv_cache_q8_desc& d, const enigma_kv_cache_rows& rows,
                              cudaStream_t s);
cudaError_t kv_cache_q8_read(const enigma_kv_cache_q8_desc& d, const enigma_kv_cache_rows& rows,
                             cudaStream_t s);
size_t sdpa_quantized_workspace(const enigma_sdpa_quantized_desc& d);
cudaError_t sdpa_quantized_launch(const enigma_sdpa_quantized_desc& d, cudaStream_t s);

cudaError_t elementwise_launch(int op, int dtype, const void* a, const void* b, void* c, int64_t n,
                               cudaStream_t s);

// Launches `kernel` as a programmatic dependent of the kernel before it on the stream: it may
// start while that one still runs, and waits (griddep_wait) before it reads what that one wrote.
template <typename... Params, typename... Args>
cudaError_t launch_dependent(void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem,
                             cudaStream_t s, Args&&... args) {
  cudaLaunchConfig_t c = {};
  c.gridDim = grid;
  c.blockDim = block;
  c.dynamicSmemBytes = smem;
  c.stream = s;
  cudaLaunchAttribute a[1];
  a[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  a[0].val.programmaticStreamSerializationAllowed = 1;
  c.attrs = a;
  c.numAttrs = 1;
  return cudaLaunchKernelEx(&c, kernel, static_cast<Params>(args)...);
}

// Records the name of the device kernel an operator launcher chose, for
// enigma_last_kernel on the calling thread (a static string).
void note_kernel(const char* name);

// Records a message for enigma_last_error on the calling thread.
void set_error(const char* fmt, ...);

}  // namespace enigma
