// pe_reduce.cu - sums of partial results over their first axis, in a fixed order.
#include "pe_mixer.cuh"

namespace pe {

namespace {

// out[c] = sum_r part[r][c]. A block has 32 columns and 8 row lanes: lane y adds the
// rows y, y + 8, ..., then the eight sums are added in order, so that the same input
// gives the same bits. Reads of a warp are 128 contiguous bytes.
template <typename T>
__global__ void __launch_bounds__(256) sum_rows_kernel(const float* __restrict__ part, int64_t rows, int64_t cols,
                                                       T* __restrict__ out) {
    __shared__ float s[8][33];
    const int x = threadIdx.x % 32, y = threadIdx.x / 32;
    for (int64_t c0 = (int64_t)blockIdx.x * 32; c0 < cols; c0 += (int64_t)gridDim.x * 32) {
        const int64_t c = c0 + x;
        float a = 0.0f;
        if (c < cols) {
#pragma unroll 4
            for (int64_t r = y; r < rows; r += 8) a += __ldg(part + r * cols + c);
        }
        s[y][x] = a;
        __syncthreads();
        if (y == 0 && c < cols) {
#pragma unroll
            for (int k = 1; k < 8; ++k) a += s[k][x];
            out[c] = from_float<T>(a);
        }
        __syncthreads();
    }
}

}  // namespace

int sum_rows(const float* part, int64_t rows, int64_t cols, int dtype, void* out, cudaStream_t s) {
    if (cols <= 0) return PE_OK;
    const int64_t blocks = ceil_div(cols, 32);
    const unsigned grid = (unsigned)(blocks < (1 << 20) ? blocks : (1 << 20));
    if (dtype == PE_F32)
        sum_rows_kernel<<<grid, 256, 0, s>>>(part, rows, cols, (float*)out);
    else if (dtype == PE_F16)
        sum_rows_kernel<<<grid, 256, 0, s>>>(part, rows, cols, (__half*)out);
    else
        sum_rows_kernel<<<grid, 256, 0, s>>>(part, rows, cols, (__nv_bfloat16*)out);
    count_launch();
    return cudaGetLastError() == cudaSuccess ? PE_OK : PE_ERR_CUDA;
}

}  // namespace pe
