// pe_reduce.cu - sums of partial results over their first axis, in a fixed order.
#include "pe_mixer.cuh"

namespace pe {

namespace {

// out[c] = sum_r part[r][c] of each job (blockIdx.y). A block has 32 columns and 32 row
// lanes: lane y adds the rows y, y + 32, ..., eight loads in flight, then the 32 sums are
// added in order, so that the same input gives the same bits. Reads of a warp are 128
// contiguous bytes. Bound by latency at the usual sizes (a few hundred rows: 4 us on a
// B200), so all of an operator's sums go in one launch.
struct Jobs {
    SumJob j[3];
};

__device__ __forceinline__ void store_sum(const SumJob& j, int64_t c, float a) {
    if (j.dtype == PE_F32)
        ((float*)j.out)[c] = a;
    else if (j.dtype == PE_F16)
        ((__half*)j.out)[c] = from_float<__half>(a);
    else
        ((__nv_bfloat16*)j.out)[c] = from_float<__nv_bfloat16>(a);
}

__global__ void __launch_bounds__(1024) sum_rows_kernel(const __grid_constant__ Jobs jobs) {
    __shared__ float s[32][33];
    const SumJob& j = jobs.j[blockIdx.y];
    const int x = threadIdx.x % 32, y = threadIdx.x / 32;
    for (int64_t c0 = (int64_t)blockIdx.x * 32; c0 < j.cols; c0 += (int64_t)gridDim.x * 32) {
        const int64_t c = c0 + x;
        float a = 0.0f;
        if (c < j.cols) {
#pragma unroll 8
            for (int64_t r = y; r < j.rows; r += 32) a += __ldg(j.part + r * j.cols + c);
        }
        s[y][x] = a;
        __syncthreads();
        if (y == 0 && c < j.cols) {
#pragma unroll
            for (int k = 1; k < 32; ++k) a += s[k][x];
            store_sum(j, c, a);
        }
        __syncthreads();
    }
}

// The same for a few rows: a thread a column, where the columns alone fill the GPU. The
// scan's training step of 2 x 256 tokens, 4096 channels and 16 states: 128 us, 140 with
// the kernel above; the norm's of 16 rows and 4096 channels, which that rule leaves to the
// kernel above: 20.7 and 16.6.
__global__ void __launch_bounds__(256) sum_few_rows(const __grid_constant__ Jobs jobs) {
    const SumJob& j = jobs.j[blockIdx.y];
    for (int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x; c < j.cols; c += (int64_t)gridDim.x * 256) {
        float a = 0.0f;
#pragma unroll 8
        for (int64_t r = 0; r < j.rows; ++r) a += __ldg(j.part + r * j.cols + c);
        store_sum(j, c, a);
    }
}

}  // namespace

int sum_rows(const SumJob* jobs, int count, cudaStream_t s) {
    Jobs all{};
    int n = 0;
    int64_t most = 0, rows = 0;
    for (int i = 0; i < count; ++i)
        if (jobs[i].out && jobs[i].cols > 0) {
            all.j[n++] = jobs[i];
            most = jobs[i].cols > most ? jobs[i].cols : most;
            rows = jobs[i].rows > rows ? jobs[i].rows : rows;
        }
    if (!n) return PE_OK;
    const bool few = rows <= 16 && ceil_div(most, 32) > 2 * num_sms();
    const int64_t blocks = ceil_div(most, few ? 256 : 32);
    const dim3 grid((unsigned)(blocks < (1 << 20) ? blocks : (1 << 20)), n);
    if (few)
        sum_few_rows<<<grid, 256, 0, s>>>(all);
    else
        sum_rows_kernel<<<grid, 1024, 0, s>>>(all);
    count_launch();
    return cudaGetLastError() == cudaSuccess ? PE_OK : PE_ERR_CUDA;
}

}  // namespace pe
