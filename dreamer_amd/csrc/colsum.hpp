// Last step of column sums: workgroups leave `slices` rows of partial sums, which are added here in a fixed order.
#pragma once
#include "elem.hpp"

namespace drm {

// 32 columns x 32 groups of slices per workgroup (short of bytes and long of latency: eight loads under way per thread; 1024 x 8192
// sums 10 us, against 90 with a thread per column), groups added in order.  Workgroups beyond 2^21 along the second axis (a launch takes
// fewer than 2^32 threads along one).  Column c < first: a[c], else b[c - first].
static __global__ __launch_bounds__(1024) void k_join_columns(const float* __restrict__ partials, int slices, int64_t cols, int64_t first, int type,
                                                              void* a, void* b) {
    __shared__ float s_part[32][33];
    const int g = threadIdx.x >> 5, l = threadIdx.x & 31;
    const int64_t c = (((int64_t)blockIdx.y << 21) + blockIdx.x) * 32 + l;
    float sum[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) sum[u] = 0.f;
    if (c < cols) {
        int s = g;
        for (; s + 7 * 32 < slices; s += 8 * 32) {
            float v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = partials[(int64_t)(s + u * 32) * cols + c];
#pragma unroll
            for (int u = 0; u < 8; ++u) sum[u] += v[u];
        }
        for (; s < slices; s += 32) sum[0] += partials[(int64_t)s * cols + c];
    }
    s_part[g][l] = ((sum[0] + sum[1]) + (sum[2] + sum[3])) + ((sum[4] + sum[5]) + (sum[6] + sum[7]));
    __syncthreads();
    if (g == 0 && c < cols) {
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < 32; ++k) v += s_part[k][l];
        if (c < first) { if (a != nullptr) store_elem(a, type, c, v); }
        else if (b != nullptr) store_elem(b, type, c - first, v);
    }
}
static inline void join_columns(const float* partials, int slices, int64_t cols, int64_t first, int type, void* a, void* b, hipStream_t s) {
    const int64_t groups = (cols + 31) / 32, row = (int64_t)1 << 21;
    k_join_columns<<<dim3((unsigned)(groups < row ? groups : row), (unsigned)((groups + row - 1) / row)), 1024, 0, s>>>(partials, slices, cols, first, type, a, b);
}

}  // namespace drm
