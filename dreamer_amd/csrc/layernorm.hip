// LayerNorm over the rows of a matrix, forward and backward with the reduction of the weight's and the bias's gradient.
//
//   m = mean(x), r = 1 / sqrt(mean((x - m)^2) + eps), xh = (x - m) r, y = xh w + b
//   dx = r (g - mean(g) - xh mean(g xh)),  g = dy w;      dw = sum over rows of dy xh;      db = sum over rows of dy
//
// Both directions are streams: forward reads x and writes y, backward reads x and dy and writes dx.  A row is held in
// registers between its statistics and its results (one wave for up to 64 x 16 elements, else one workgroup), so that x is
// read once and the variance is taken about the mean.  Workgroups walk over rows: the weight and the bias stay in registers
// for all of them, and so do the column sums of the backward pass, which go to `partials` once per workgroup and are added
// there in a fixed order (no atomics: results do not depend on the order in which workgroups run).
#include "elem.hpp"

#include <type_traits>

namespace drm {

// sums of two values over the TPB threads that share a row; every thread receives them.  `buf` alternates between calls so
// that one barrier per call is enough.
template <int TPB>
__device__ __forceinline__ void row_sum2(float& a, float& b, float (*buf)[2]) {
    a = group_sum<64>(a);
    b = group_sum<64>(b);
    if constexpr (TPB > 64) {
        constexpr int W = TPB / 64;
        const int w = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) { buf[w][0] = a; buf[w][1] = b; }
        __syncthreads();
        a = 0.f; b = 0.f;
#pragma unroll
        for (int i = 0; i < W; ++i) { a += buf[i][0]; b += buf[i][1]; }
    }
}
template <int TPB>
__device__ __forceinline__ float row_sum(float a, float (*buf)[2]) {
    float z = 0.f;
    row_sum2<TPB>(a, z, buf);
    return a;
}

// TPB threads per row; 64: four rows per workgroup, one per wave
template <typename T, int TPB, int CH>
__global__ __launch_bounds__(TPB == 64 ? 256 : TPB) void k_norm_fwd(const T* __restrict__ x, int64_t ldx, const void* w, const void* b,
                                                                    int wtype, T* __restrict__ y, int64_t ldy,
                                                                    float* __restrict__ mean, float* __restrict__ rstd, int64_t N,
                                                                    int E, float eps) {
    constexpr int VEC = Elem<T>::VEC, RPB = TPB == 64 ? 4 : 1;
    __shared__ float s_buf[2][TPB / 64][2];
    const int t = TPB == 64 ? (threadIdx.x & 63) : threadIdx.x;
    float wv[CH][VEC], bv[CH][VEC];
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const int e = (c * TPB + t) * VEC + i;
            wv[c][i] = w != nullptr && e < E ? load_elem(w, wtype, e) : 1.f;
            bv[c][i] = b != nullptr && e < E ? load_elem(b, wtype, e) : 0.f;
        }
    const float inv = 1.f / (float)E;
    for (int64_t n = (int64_t)blockIdx.x * RPB + (TPB == 64 ? threadIdx.x >> 6 : 0); n < N; n += (int64_t)gridDim.x * RPB) {
        const T* row = x + n * ldx;
        float v[CH][VEC], s = 0.f;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            load_slot(row, (int64_t)(c * TPB + t) * VEC, E, 0.f, v[c]);
#pragma unroll
            for (int i = 0; i < VEC; ++i) s += v[c][i];
        }
        const float m = row_sum<TPB>(s, s_buf[0]) * inv;
        float q = 0.f;
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                v[c][i] -= m;
                if ((c * TPB + t) * VEC + i < E) q += v[c][i] * v[c][i];
            }
        const float r = 1.f / sqrtf(row_sum<TPB>(q, s_buf[1]) * inv + eps);
        if (t == 0 && mean != nullptr) { mean[n] = m; rstd[n] = r; }
        T* out = y + n * ldy;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[c][i] = fmaf(v[c][i] * r, wv[c][i], bv[c][i]);
            store_slot(out, (int64_t)(c * TPB + t) * VEC, E, v[c]);
        }
    }
}

// Rows too long for registers: three walks over the row (the second and third find it in the caches unless it is longer than
// those).  One workgroup per row.
template <typename T>
__global__ __launch_bounds__(1024) void k_norm_fwd_long(const T* __restrict__ x, int64_t ldx, const void* w, const void* b, int wtype,
                                                        T* __restrict__ y, int64_t ldy, float* __restrict__ mean,
                                                        float* __restrict__ rstd, int64_t N, int E, float eps) {
    constexpr int VEC = Elem<T>::VEC;
    __shared__ float s_buf[2][16][2];
    const float inv = 1.f / (float)E;
    for (int64_t n = blockIdx.x; n < N; n += gridDim.x) {
        const T* row = x + n * ldx;
        float v[VEC], s = 0.f, q = 0.f;
        for (int64_t e = (int64_t)threadIdx.x * VEC; e < E; e += 1024 * VEC) {
            load_slot(row, e, E, 0.f, v);
            float p = 0.f;
#pragma unroll
            for (int i = 0; i < VEC; ++i) p += v[i];
            s += p;
        }
        const float m = row_sum<1024>(s, s_buf[0]) * inv;
        for (int64_t e = (int64_t)threadIdx.x * VEC; e < E; e += 1024 * VEC) {
            load_slot(row, e, E, m, v);
            float p = 0.f;
#pragma unroll
            for (int i = 0; i < VEC; ++i) p += (v[i] - m) * (v[i] - m);
            q += p;
        }
        const float r = 1.f / sqrtf(row_sum<1024>(q, s_buf[1]) * inv + eps);
        if (threadIdx.x == 0 && mean != nullptr) { mean[n] = m; rstd[n] = r; }
        for (int64_t e = (int64_t)threadIdx.x * VEC; e < E; e += 1024 * VEC) {
            load_slot(row, e, E, 0.f, v);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const int64_t k = min(e + i, (int64_t)E - 1);
                v[i] = fmaf((v[i] - m) * r, w != nullptr ? load_elem(w, wtype, k) : 1.f, b != nullptr ? load_elem(b, wtype, k) : 0.f);
            }
            store_slot(y + n * ldy, e, E, v);
        }
    }
}

// partials: (gridDim.x, 2, E): column sums of dy xh and of dy over the rows this workgroup walked
template <typename T, int TPB, int CH>
__global__ __launch_bounds__(TPB == 64 ? 256 : TPB) void k_norm_bwd(const T* __restrict__ x, int64_t ldx, const T* __restrict__ dy,
                                                                    int64_t lddy, const void* w, int wtype,
                                                                    const float* __restrict__ mean, const float* __restrict__ rstd,
                                                                    T* __restrict__ dx, float* __restrict__ partials, int64_t N,
                                                                    int E) {
    constexpr int VEC = Elem<T>::VEC, RPB = TPB == 64 ? 4 : 1;
    __shared__ float s_buf[2][TPB / 64][2];
    __shared__ float s_cols[TPB == 64 ? 64 * CH * VEC : 1];
    const int t = TPB == 64 ? (threadIdx.x & 63) : threadIdx.x;
    float wv[CH][VEC], aw[CH][VEC], ab[CH][VEC];
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const int e = (c * TPB + t) * VEC + i;
            wv[c][i] = w != nullptr && e < E ? load_elem(w, wtype, e) : 1.f;
            aw[c][i] = 0.f;
            ab[c][i] = 0.f;
        }
    const float inv = 1.f / (float)E;
    int flip = 0;
    for (int64_t n = (int64_t)blockIdx.x * RPB + (TPB == 64 ? threadIdx.x >> 6 : 0); n < N; n += (int64_t)gridDim.x * RPB, flip ^= 1) {
        const float m = mean[n], r = rstd[n];
        float xh[CH][VEC], g[CH][VEC], s = 0.f, q = 0.f;
#pragma unroll
        for (int c = 0; c < CH; ++c) load_slot(x + n * ldx, (int64_t)(c * TPB + t) * VEC, E, m, xh[c]);   // beyond the row: xh = 0
#pragma unroll
        for (int c = 0; c < CH; ++c) load_slot(dy + n * lddy, (int64_t)(c * TPB + t) * VEC, E, 0.f, g[c]);
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float h = (xh[c][i] - m) * r, d = g[c][i];
                aw[c][i] = fmaf(d, h, aw[c][i]);
                ab[c][i] += d;
                const float gw = d * wv[c][i];
                s += gw;
                q = fmaf(gw, h, q);
                xh[c][i] = h;
                g[c][i] = gw;
            }
        row_sum2<TPB>(s, q, s_buf[flip]);
        if (dx != nullptr) {
            s *= inv; q *= inv;
#pragma unroll
            for (int c = 0; c < CH; ++c) {
#pragma unroll
                for (int i = 0; i < VEC; ++i) g[c][i] = r * (g[c][i] - fmaf(xh[c][i], q, s));
                store_slot(dx + n * (int64_t)E, (int64_t)(c * TPB + t) * VEC, E, g[c]);
            }
        }
    }
    if (partials == nullptr) return;
    float* pw = partials + (int64_t)blockIdx.x * 2 * E;
    if constexpr (TPB == 64) {   // the four waves' sums, one wave after the other
        const int wave = threadIdx.x >> 6;
#pragma unroll
        for (int half = 0; half < 2; ++half)
            for (int k = 0; k < 4; ++k) {
                __syncthreads();
                if (wave != k) continue;
#pragma unroll
                for (int c = 0; c < CH; ++c)
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        const int e = (c * TPB + t) * VEC + i;
                        const float mine = half == 0 ? aw[c][i] : ab[c][i];
                        const float sum = (k == 0 ? 0.f : s_cols[e]) + mine;
                        if (k < 3) s_cols[e] = sum;
                        else if (e < E) pw[(int64_t)half * E + e] = sum;
                    }
            }
    } else {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
#pragma unroll
            for (int h = 0; h < VEC; h += 4) {
                const float a[4] = {aw[c][h], aw[c][h + 1], aw[c][h + 2], aw[c][h + 3]};
                const float b[4] = {ab[c][h], ab[c][h + 1], ab[c][h + 2], ab[c][h + 3]};
                store_slot(pw, (int64_t)(c * TPB + t) * VEC + h, E, a);
                store_slot(pw + E, (int64_t)(c * TPB + t) * VEC + h, E, b);
            }
        }
    }
}

// rows too long for registers: the two row means first ...
template <typename T>
__global__ __launch_bounds__(1024) void k_norm_bwd_sums(const T* __restrict__ x, int64_t ldx, const T* __restrict__ dy, int64_t lddy,
                                                        const void* w, int wtype, const float* __restrict__ mean,
                                                        const float* __restrict__ rstd, float* __restrict__ sums, int64_t N, int E) {
    constexpr int VEC = Elem<T>::VEC;
    __shared__ float s_buf[2][16][2];
    int flip = 0;
    for (int64_t n = blockIdx.x; n < N; n += gridDim.x, flip ^= 1) {
        const float m = mean[n], r = rstd[n];
        float xv[VEC], g[VEC], s = 0.f, q = 0.f;
        for (int64_t e = (int64_t)threadIdx.x * VEC; e < E; e += 1024 * VEC) {
            load_slot(x + n * ldx, e, E, m, xv);
            load_slot(dy + n * lddy, e, E, 0.f, g);
            float ps = 0.f, pq = 0.f;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float gw = g[i] * (w != nullptr ? load_elem(w, wtype, min(e + i, (int64_t)E - 1)) : 1.f);
                ps += gw;
                pq = fmaf(gw, (xv[i] - m) * r, pq);
            }
            s += ps; q += pq;
        }
        row_sum2<1024>(s, q, s_buf[flip]);
        if (threadIdx.x == 0) { sums[2 * n] = s / (float)E; sums[2 * n + 1] = q / (float)E; }
    }
}
// ... then a strip of columns over a slice of the rows: dx and the column sums (blockIdx.x: strip, blockIdx.y: slice)
template <typename T>
__global__ __launch_bounds__(256) void k_norm_bwd_cols(const T* __restrict__ x, int64_t ldx, const T* __restrict__ dy, int64_t lddy,
                                                       const void* w, int wtype, const float* __restrict__ mean,
                                                       const float* __restrict__ rstd, const float* __restrict__ sums,
                                                       T* __restrict__ dx, float* __restrict__ partials, int64_t N, int E) {
    constexpr int VEC = Elem<T>::VEC;
    const int64_t e = ((int64_t)blockIdx.x * 256 + threadIdx.x) * VEC;
    if (e >= E) return;
    float wv[VEC], aw[VEC], ab[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        wv[i] = w != nullptr ? load_elem(w, wtype, min(e + i, (int64_t)E - 1)) : 1.f;
        aw[i] = 0.f;
        ab[i] = 0.f;
    }
    for (int64_t n = blockIdx.y; n < N; n += gridDim.y) {
        const float m = mean[n], r = rstd[n];
        float xv[VEC], g[VEC];
        load_slot(x + n * ldx, e, E, m, xv);
        load_slot(dy + n * lddy, e, E, 0.f, g);
        const float s = sums != nullptr ? sums[2 * n] : 0.f, q = sums != nullptr ? sums[2 * n + 1] : 0.f;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const float h = (xv[i] - m) * r;
            aw[i] = fmaf(g[i], h, aw[i]);
            ab[i] += g[i];
            g[i] = r * (g[i] * wv[i] - fmaf(h, q, s));
        }
        if (dx != nullptr) store_slot(dx + n * (int64_t)E, e, E, g);
    }
    if (partials != nullptr) {
        float* pw = partials + (int64_t)blockIdx.y * 2 * E;
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            if (e + i < E) { pw[e + i] = aw[i]; pw[E + e + i] = ab[i]; }
    }
}

// Column sums over the slices: 64 columns x 4 slice groups per workgroup, groups added in order.  Column c < E: dw, else db.
__global__ __launch_bounds__(256) void k_norm_cols(const float* __restrict__ partials, int slices, int E, int wtype, void* dw, void* db) {
    __shared__ float s_part[4][64];
    const int g = threadIdx.x >> 6, l = threadIdx.x & 63;
    const int64_t c = (int64_t)blockIdx.x * 64 + l, cols = 2 * (int64_t)E;
    float a0 = 0.f, a1 = 0.f, a2 = 0.f, a3 = 0.f;
    if (c < cols) {
        int s = g;
        for (; s + 12 < slices; s += 16) {
            a0 += partials[(int64_t)s * cols + c];
            a1 += partials[(int64_t)(s + 4) * cols + c];
            a2 += partials[(int64_t)(s + 8) * cols + c];
            a3 += partials[(int64_t)(s + 12) * cols + c];
        }
        for (; s < slices; s += 4) a0 += partials[(int64_t)s * cols + c];
    }
    s_part[g][l] = (a0 + a1) + (a2 + a3);
    __syncthreads();
    if (g == 0 && c < cols) {
        const float v = (s_part[0][l] + s_part[1][l]) + (s_part[2][l] + s_part[3][l]);
        if (c < E) { if (dw != nullptr) store_elem(dw, wtype, c, v); }
        else if (db != nullptr) store_elem(db, wtype, c - E, v);
    }
}

// ---- host side -------------------------------------------------------------------------------------------------------
// Threads per row by the row's length: enough for 16 elements a thread (16 values, weights and two running column sums fit
// the registers at four waves per SIMD).
constexpr int NORM_MAX_E = 1024 * 16;
static inline int norm_threads(int E) { return E <= 1024 ? 64 : E <= 4096 ? 256 : E <= 8192 ? 512 : 1024; }
// workgroups that walk the rows
static inline int norm_slices(int64_t N, int E) {
    if (E > NORM_MAX_E) return (int)(N < 64 ? (N > 0 ? N : 1) : 64);
    const int tpb = norm_threads(E);
    const int64_t rows = tpb == 64 ? (N + 3) / 4 : N, cap = 512;
    return (int)(rows < 1 ? 1 : rows < cap ? rows : cap);
}

template <typename T, typename F>
static int norm_variant(int E, F&& f) {
    constexpr int VEC = Elem<T>::VEC, C8 = 8 / VEC, C16 = 16 / VEC;
#define DRM_NORM_CASE(TPB, CH) return f(std::integral_constant<int, TPB>{}, std::integral_constant<int, CH>{})
    if (E <= 64 * VEC) DRM_NORM_CASE(64, 1);
    if (E <= 512) DRM_NORM_CASE(64, C8);
    if (E <= 1024) DRM_NORM_CASE(64, C16);
    if (E <= 2048) DRM_NORM_CASE(256, C8);
    if (E <= 4096) DRM_NORM_CASE(256, C16);
    if (E <= 8192) DRM_NORM_CASE(512, C16);
    DRM_NORM_CASE(1024, C16);
#undef DRM_NORM_CASE
}

static int norm_check(const char* what, const void* x, int64_t ldx, int x_dtype, int w_dtype, int64_t N, int32_t E) {
    DRM_REQUIRE(x, DRM_EINVAL, "%s: null pointer", what);
    DRM_REQUIRE(elem_ok(x_dtype) && (w_dtype == DRM_F32 || w_dtype == x_dtype), DRM_ENOTSUP,
                "%s: element types %d / %d (rows fp32, bf16 or fp16; weights fp32 or the rows' type)", what, x_dtype, w_dtype);
    DRM_REQUIRE(N >= 0 && E >= 1 && ldx >= E, DRM_EINVAL, "%s: N=%lld E=%d row stride %lld", what, (long long)N, E, (long long)ldx);
    return DRM_OK;
}

}  // namespace drm

using namespace drm;

extern "C" int drm_layer_norm_forward(const void* x, int64_t ldx, int32_t x_dtype, const void* w, const void* b, int32_t w_dtype,
                                      void* y, int64_t ldy, float* mean, float* rstd, int64_t N, int32_t E, float eps,
                                      drm_stream_t stream) {
    if (N == 0 && E >= 1) return DRM_OK;
    if (int rc = norm_check(__func__, x, ldx, x_dtype, w_dtype, N, E)) return rc;
    DRM_REQUIRE(y && ldy >= E, DRM_EINVAL, "null output or row stride %lld below E=%d", (long long)ldy, E);
    DRM_REQUIRE((mean == nullptr) == (rstd == nullptr), DRM_EINVAL, "mean and rstd are saved together");
    hipStream_t s = (hipStream_t)stream;
    const double n = (double)N * E;
    ProfScope ps(PC_ELEMENTWISE, s, 8 * n, 2 * n * elem_bytes(x_dtype));
    return with_elem(x_dtype, [&](auto tag) -> int {
        using T = decltype(tag);
        if (E > NORM_MAX_E) {
            k_norm_fwd_long<T><<<(int)(N < 2048 ? N : 2048), 1024, 0, s>>>((const T*)x, ldx, w, b, w_dtype, (T*)y, ldy, mean, rstd, N, E, eps);
        } else {
            norm_variant<T>(E, [&](auto tpb, auto ch) {
                constexpr int TPB = decltype(tpb)::value, CH = decltype(ch)::value;
                const int64_t rows = TPB == 64 ? (N + 3) / 4 : N;
                const int grid = (int)(rows < 2048 ? rows : 2048);
                k_norm_fwd<T, TPB, CH><<<grid, TPB == 64 ? 256 : TPB, 0, s>>>((const T*)x, ldx, w, b, w_dtype, (T*)y, ldy, mean, rstd, N, E, eps);
                return 0;
            });
        }
        DRM_LAUNCH_CHECK();
        return DRM_OK;
    });
}

extern "C" size_t drm_layer_norm_workspace_bytes(int64_t N, int32_t E) {
    if (N < 0 || E < 1) return 0;
    const size_t sums = E > NORM_MAX_E ? (size_t)N * 2 * sizeof(float) : 0;
    return sums + (size_t)norm_slices(N, E) * 2 * E * sizeof(float);
}

extern "C" int drm_layer_norm_backward(const void* x, int64_t ldx, const void* dy, int64_t lddy, int32_t x_dtype, const void* w,
                                       int32_t w_dtype, const float* mean, const float* rstd, void* dx, void* dw, void* db,
                                       int64_t N, int32_t E, void* workspace, size_t workspace_bytes, drm_stream_t stream) {
    hipStream_t s = (hipStream_t)stream;
    const bool cols = dw != nullptr || db != nullptr;
    DRM_REQUIRE(N >= 0 && E >= 1, DRM_EINVAL, "N=%lld E=%d", (long long)N, E);
    DRM_REQUIRE(elem_ok(x_dtype) && (w_dtype == DRM_F32 || w_dtype == x_dtype), DRM_ENOTSUP, "element types %d / %d", x_dtype, w_dtype);
    const int cgrid = (int)((2 * (int64_t)E + 63) / 64);
    if (N == 0) {
        if (cols) { k_norm_cols<<<cgrid, 256, 0, s>>>(nullptr, 0, E, w_dtype, dw, db); DRM_LAUNCH_CHECK(); }
        return DRM_OK;
    }
    if (int rc = norm_check(__func__, x, ldx, x_dtype, w_dtype, N, E)) return rc;
    DRM_REQUIRE(dy && lddy >= E && mean && rstd, DRM_EINVAL, "null pointer or row stride %lld below E=%d", (long long)lddy, E);
    if (!dx && !cols) return DRM_OK;
    DRM_REQUIRE(workspace && workspace_bytes >= drm_layer_norm_workspace_bytes(N, E), DRM_EINVAL, "workspace of %zu bytes, %zu needed",
                workspace ? workspace_bytes : (size_t)0, drm_layer_norm_workspace_bytes(N, E));
    const int slices = norm_slices(N, E);
    const double n = (double)N * E;
    ProfScope ps(PC_ELEMENTWISE, s, 17 * n, 3 * n * elem_bytes(x_dtype));
    float* sums = (float*)workspace;
    float* part = !cols ? nullptr : E > NORM_MAX_E ? sums + 2 * N : sums;
    const int rc = with_elem(x_dtype, [&](auto tag) -> int {
        using T = decltype(tag);
        if (E > NORM_MAX_E) {
            if (dx != nullptr) {
                k_norm_bwd_sums<T><<<(int)(N < 2048 ? N : 2048), 1024, 0, s>>>((const T*)x, ldx, (const T*)dy, lddy, w, w_dtype, mean, rstd, sums, N, E);
                DRM_LAUNCH_CHECK();
            }
            constexpr int STRIP = 256 * Elem<T>::VEC;
            k_norm_bwd_cols<T><<<dim3((unsigned)(((int64_t)E + STRIP - 1) / STRIP), slices), 256, 0, s>>>((const T*)x, ldx, (const T*)dy, lddy, w, w_dtype, mean, rstd,
                                                                                      dx != nullptr ? sums : nullptr, (T*)dx, part, N, E);
        } else {
            norm_variant<T>(E, [&](auto tpb, auto ch) {
                constexpr int TPB = decltype(tpb)::value, CH = decltype(ch)::value;
                k_norm_bwd<T, TPB, CH><<<slices, TPB == 64 ? 256 : TPB, 0, s>>>((const T*)x, ldx, (const T*)dy, lddy, w, w_dtype, mean, rstd, (T*)dx, part, N, E);
                return 0;
            });
        }
        DRM_LAUNCH_CHECK();
        return DRM_OK;
    });
    if (rc != DRM_OK || !cols) return rc;
    k_norm_cols<<<cgrid, 256, 0, s>>>(part, slices, E, w_dtype, dw, db);
    DRM_LAUNCH_CHECK();
    return DRM_OK;
}
