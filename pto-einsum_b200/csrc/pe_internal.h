// pe_internal.h - declarations shared between the core library's translation units.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "pto_einsum_b200.h"

namespace pe {

int set_last_error(int code);
int check_cuda(cudaError_t e);
int num_sms();
void count_launch(int n = 1);

int elementwise_mul(int32_t dtype, const void* a, const void* b, float* out, int64_t n,
                    cudaStream_t s);
int broadcast_mul(const pe_broadcast_plan* pl, const void* full, const void* bc, float* out,
                  cudaStream_t s);
int permute(const pe_permute_plan* pl, const void* in, void* out, cudaStream_t s);

// Generic strided copy over a logical index space (outermost axis first).
int strided_copy_launch(int es, int nd, const int64_t* size, const int64_t* sst,
                        const int64_t* dst_st, const void* src, void* dst, cudaStream_t s);

int contract_workspace_bytes(const pe_contract_plan* plan, size_t* bytes);
// Scratch bytes pe_contract needs for these exact input pointers.
int contract_scratch_bytes(const pe_contract_plan* plan, const void* in0, const void* in1, size_t* bytes);
int contract(const pe_contract_plan* plan, const void* in0, const void* in1, float* out, void* ws,
             size_t ws_bytes, cudaStream_t s);

// Prepared-launch cache held by a workspace handle: contract_cached replays the
// launches of an earlier call with the same plan object and pointers.
void* program_cache_create();
void program_cache_destroy(void* cache);
// phase: EINSUM_PHASE_STOP level (3 = the full contraction)
int contract_cached(void* cache, const pe_contract_plan* plan, const void* in0, const void* in1, float* out,
                    void* ws, size_t ws_bytes, int phase, cudaStream_t s);

// Read (and optionally clear) the device error word of the GEMM kernels.
int gemm_device_error(bool clear);
int wait_timeout_selftest(uint64_t timeout_ns, cudaStream_t s);

// out[c] = sum over r < rows of part[r][c], rounded to dtype, in a fixed order of
// additions; up to three at once, those without an `out` left out.
struct SumJob {
    const float* part;
    int64_t rows, cols;
    int dtype;
    void* out;
};
int sum_rows(const SumJob* jobs, int count, cudaStream_t s);

// Recurrent-mixer operators.
int64_t scan_ckpt_floats(int64_t tokens, int64_t nseq, int64_t packed, int64_t channels, int64_t states);
int64_t scan_ws_bytes(const pe_scan_args* a);
int selective_scan(const pe_scan_args* a, cudaStream_t s);
int64_t scan_grad_ws_bytes(const pe_scan_grad_args* a);
int selective_scan_grad(const pe_scan_grad_args* a, cudaStream_t s);
int selective_scan_step(const pe_scan_step_args* a, cudaStream_t s);
int scan_device_error(bool clear);
int scan_grad_device_error(bool clear);
int causal_conv(const pe_conv_args* a, cudaStream_t s);
int64_t conv_grad_ws_bytes(const pe_conv_grad_args* a);
int causal_conv_grad(const pe_conv_grad_args* a, cudaStream_t s);
int causal_conv_step(const pe_conv_step_args* a, cudaStream_t s);
int conv_device_error(bool clear);
int64_t norm_ws_bytes(const pe_norm_args* a);
int group_norm(const pe_norm_args* a, cudaStream_t s);
int64_t norm_grad_ws_bytes(const pe_norm_grad_args* a);
int group_norm_grad(const pe_norm_grad_args* a, cudaStream_t s);

}  // namespace pe
