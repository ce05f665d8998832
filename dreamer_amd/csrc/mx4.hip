// Microscaled 4-bit floating point: quantisation, its inverse, and the products that read 4-bit weights.
#include "mx4.hpp"

#include <climits>

namespace drm {

// ---- quantisation -------------------------------------------------------------------------------------------------------
// e = floor(log2(max |x|)) - 2, clamped to [-127, 127]; code = x / 2^e rounded to the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6 (ties
// to the even code), 6 beyond.  Four lanes share a block: eight elements, four code bytes each.  A stream: bound by the bytes.
template <typename T>
__global__ __launch_bounds__(256) void k_mx4_quantize(const T* __restrict__ x, int64_t ldx, int64_t rows, int K, int nb,
                                                      uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    const int64_t quads = rows * nb * 4, step = (int64_t)gridDim.x * 256;
    for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < quads; q += step) {   // quads of a block stay in one wave
        const int64_t blk = q >> 2, r = blk / nb;
        const int64_t at = (blk - r * nb) * 32 + (q & 3) * 8;
        const T* row = x + r * ldx;
        float v[8];
        if constexpr (Elem<T>::VEC == 8) {
            load_slot(row, at, K, 0.f, v);
        } else {
            float a[4], b[4];
            load_slot(row, at, K, 0.f, a);
            load_slot(row, at + 4, K, 0.f, b);
#pragma unroll
            for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[i + 4] = b[i]; }
        }
        // as integers the magnitudes order like the values, and infinities and NaN come out on top
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, __builtin_bit_cast(uint32_t, v[i]) & 0x7fffffffu);
        top = max(top, (uint32_t)xor_lane_i<1>((int)top));
        top = max(top, (uint32_t)xor_lane_i<2>((int)top));
        const int ex = (int)(top >> 23);                 // biased exponent; 0: below 2^-126
        const int s = ex == 255 ? 255 : max(ex - 2, 0);
        uint32_t out = 0;
        if (s != 255) {
            // 2^-e = 2^(127 - s), s <= 252; the products are exact unless they are far below the smallest code's half
            const float inv = __builtin_bit_cast(float, (uint32_t)(254 - s) << 23);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] *= inv;
            out = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(out, v[0], v[1], 1.f, 0);
            out = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(out, v[2], v[3], 1.f, 1);
            out = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(out, v[4], v[5], 1.f, 2);
            out = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(out, v[6], v[7], 1.f, 3);
        }
        reinterpret_cast<uint32_t*>(codes)[q] = out;
        if ((q & 3) == 0) scales[blk] = (uint8_t)s;
    }
}

template <typename T>
__global__ __launch_bounds__(256) void k_mx4_dequantize(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int64_t rows,
                                                        int K, int nb, T* __restrict__ y, int64_t ldy) {
    const int64_t quads = rows * nb * 4, step = (int64_t)gridDim.x * 256;
    for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < quads; q += step) {
        const int64_t blk = q >> 2, r = blk / nb;
        const int64_t at = (blk - r * nb) * 32 + (q & 3) * 8;
        const uint32_t c = reinterpret_cast<const uint32_t*>(codes)[q];
        const uint32_t s = scales[blk];
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            // e2m1 as an integer: magnitudes 0, 1, 2, 3, 4, 6, 8, 12 halves
            const uint32_t m = (c >> (4 * i)) & 7u;
            const float h = (float)(m < 2 ? m : (2u | (m & 1u)) << ((m >> 1) - 1));
            const float a = s == 255u ? __builtin_bit_cast(float, 0x7fc00000u) : ldexpf(h, (int)s - 128);
            v[i] = (c >> (4 * i)) & 8u ? -a : a;
        }
        T* row = y + r * ldy;
        if constexpr (Elem<T>::VEC == 8) {
            store_slot(row, at, K, v);
        } else {
            const float a[4] = {v[0], v[1], v[2], v[3]}, b[4] = {v[4], v[5], v[6], v[7]};
            store_slot(row, at, K, a);
            store_slot(row, at + 4, K, b);
        }
    }
}

// ---- y = x W^T + bias, few rows -----------------------------------------------------------------------------------------
// The weight is streamed once: a workgroup takes 16 weight rows, its waves split the blocks.  A lane holds one block of one
// weight row (16 bytes, one scale) and feeds it to four matrix instructions, eight elements each; the four lane groups of an
// instruction hold four different blocks, which is a permutation of the reduction index that the x operand follows.
template <typename T, int MT, int NW>
__global__ __launch_bounds__(NW * 64) void k_mx4_rows(const T* __restrict__ x, int64_t ldx, Mx4 W, const void* bias, int btype,
                                                      T* __restrict__ y, int64_t ldy, int M, int K) {
    constexpr int P = Parts<T>::N;
    __shared__ f32x4 s_acc[NW][MT][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, g = lane >> 4, c = lane & 15;
    const int n0 = blockIdx.x * 16;
    const int64_t n = min(n0 + c, W.rows - 1);
    f32x4 acc[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int base = w * 4; base < W.nb; base += NW * 4) {
        const int kb = base + g;
        const bool live = kb < W.nb;
        u32x4 q{0, 0, 0, 0};
        float sc = 1.f;
        if (live) {
            q = *reinterpret_cast<const u32x4*>(W.codes + (n * W.nb + kb) * 16);
            sc = mx4_scale(W.scales[n * W.nb + kb]);
        }
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const bf16x8 a = mx4_bf16x8(q[s], sc);
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                bf16x8 b[P];
                load_parts(x + (int64_t)min(t * 16 + c, M - 1) * ldx, (int64_t)kb * 32 + s * 8, K, b);
#pragma unroll
                for (int p = P - 1; p >= 0; --p) acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b[p], acc[t], 0, 0, 0);
            }
        }
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) s_acc[w][t][lane] = acc[t];
    __syncthreads();
    for (int o = threadIdx.x; o < MT * 64; o += NW * 64) {
        const int t = o >> 6, l = o & 63;
        f32x4 v = s_acc[0][t][l];
#pragma unroll
        for (int k = 1; k < NW; ++k) v += s_acc[k][t][l];
        const int m = t * 16 + (l & 15), nn = n0 + 4 * (l >> 4);
        if (m < M)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (nn + i < W.rows) y[m * ldy + nn + i] = (T)(v[i] + (bias != nullptr ? load_elem(bias, btype, nn + i) : 0.f));
    }
}

// ---- y = x W^T + bias and dx = dy W, many rows --------------------------------------------------------------------------
// 128 x 128 output tile, reduction in steps of 64; the 4-bit operand is widened to bf16 on its way into LDS (for dx: transposed),
// the float operand goes there in its bf16 parts.  LDS rows of 64 elements = 8 chunks of 16 bytes, chunk c of row r at c ^ (r & 7).
template <typename T, bool GRAD>
__global__ __launch_bounds__(256) void k_mx4_tile(const T* __restrict__ x, int64_t ldx, Mx4 W, const void* bias, int btype,
                                                  T* __restrict__ y, int64_t ldy, int M, int N, int K) {
    // forward: reduction over W's columns (K), output columns are W's rows; gradient: the other way round (N = output columns)
    constexpr int P = Parts<T>::N, BK = 64;
    __shared__ __attribute__((aligned(16))) uint16_t s_x[P][128 * BK];
    __shared__ __attribute__((aligned(16))) uint16_t s_w[128 * BK];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int m0 = blockIdx.y * 128, n0 = blockIdx.x * 128, wm = (w >> 1) * 64, wn = (w & 1) * 64;
    f32x16 acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    for (int k0 = 0; k0 < K; k0 += BK) {
        __syncthreads();
        for (int o = threadIdx.x; o < 128 * 8; o += 256) {
            const int r = o >> 3, ch = o & 7;
            bf16x8 p[P];
            load_parts(x + (int64_t)min(m0 + r, M - 1) * ldx, k0 + ch * 8, K, p);
#pragma unroll
            for (int q = 0; q < P; ++q) *reinterpret_cast<bf16x8*>(&s_x[q][r * BK + ((ch ^ (r & 7)) * 8)]) = p[q];
        }
        if constexpr (!GRAD) {
            for (int o = threadIdx.x; o < 128 * 8; o += 256) {
                const int r = o >> 3, ch = o & 7, kb = (k0 >> 5) + (ch >> 2);
                const int64_t n = min(n0 + r, N - 1);
                bf16x8 v = mx4_bf16x8(0u, 1.f);
                if (kb < W.nb)
                    v = mx4_bf16x8(reinterpret_cast<const uint32_t*>(W.codes)[(n * W.nb + kb) * 4 + (ch & 3)], mx4_scale(W.scales[n * W.nb + kb]));
                *reinterpret_cast<bf16x8*>(&s_w[r * BK + ((ch ^ (r & 7)) * 8)]) = v;
            }
        } else {
            // eight codes of one weight row (columns n0 + ...) per step, scattered down a column of the tile
            for (int o = threadIdx.x; o < 64 * 16; o += 256) {
                const int rr = o >> 4, c8 = o & 15, col = n0 + c8 * 8, kb = col >> 5;
                const int64_t n = k0 + rr;
                bf16x8 v = mx4_bf16x8(0u, 1.f);
                if (n < W.rows && kb < W.nb)
                    v = mx4_bf16x8(reinterpret_cast<const uint32_t*>(W.codes)[(n * W.nb + kb) * 4 + ((col >> 3) & 3)], mx4_scale(W.scales[n * W.nb + kb]));
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int r = c8 * 8 + i;
                    s_w[r * BK + (((rr >> 3) ^ (r & 7)) * 8) + (rr & 7)] = __builtin_bit_cast(uint16_t, (__bf16)v[i]);
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int s = 0; s < BK / 16; ++s) {
            bf16x8 a[2], b[2];
            const int ch = s * 2 + (lane >> 5);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = wn + i * 32 + (lane & 31);
                a[i] = *reinterpret_cast<const bf16x8*>(&s_w[r * BK + ((ch ^ (r & 7)) * 8)]);
            }
#pragma unroll
            for (int p = P - 1; p >= 0; --p) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int r = wm + j * 32 + (lane & 31);
                    b[j] = *reinterpret_cast<const bf16x8*>(&s_x[p][r * BK + ((ch ^ (r & 7)) * 8)]);
                }
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[i], b[j], acc[i][j], 0, 0, 0);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int m = m0 + wm + j * 32 + (lane & 31);
            if (m >= M) continue;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int n = n0 + wn + i * 32 + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3);
                if (n < N) y[m * ldy + n] = (T)(acc[i][j][e] + (bias != nullptr ? load_elem(bias, btype, n) : 0.f));
            }
        }
}

// ---- both operands in 4 bits ----------------------------------------------------------------------------------------------
// One scaled matrix instruction takes a 16-byte block and its scale byte per lane from either operand: 16 x 16 outputs, 128 deep.
template <typename T>
__global__ __launch_bounds__(256) void k_mx4_product(Mx4 X, Mx4 W, const void* bias, int btype, T* __restrict__ y, int64_t ldy) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, g = lane >> 4, c = lane & 15;
    const int m0 = blockIdx.y * 64 + (w >> 1) * 32, n0 = blockIdx.x * 64 + (w & 1) * 32;
    f32x4 acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int base = 0; base < W.nb; base += 4) {
        const int kb = base + g;
        const bool live = kb < W.nb;
        i32x8 a[2], b[2];
        int sa[2], sb[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int64_t n = (int64_t)min(n0 + i * 16 + c, W.rows - 1) * W.nb + kb, m = (int64_t)min(m0 + i * 16 + c, X.rows - 1) * X.nb + kb;
            u32x4 qa{0, 0, 0, 0}, qb{0, 0, 0, 0};
            sa[i] = sb[i] = 127;
            if (live) {
                qa = reinterpret_cast<const u32x4*>(W.codes)[n];
                qb = reinterpret_cast<const u32x4*>(X.codes)[m];
                sa[i] = W.scales[n];
                sb[i] = X.scales[m];
            }
            a[i] = i32x8{(int)qa[0], (int)qa[1], (int)qa[2], (int)qa[3], 0, 0, 0, 0};
            b[i] = i32x8{(int)qb[0], (int)qb[1], (int)qb[2], (int)qb[3], 0, 0, 0, 0};
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a[i], b[j], acc[i][j], 4, 4, 0, sa[i], 0, sb[j]);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int m = m0 + j * 16 + c;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int n = n0 + i * 16 + 4 * g + e;
                if (m < X.rows && n < W.rows) y[m * ldy + n] = (T)(acc[i][j][e] + (bias != nullptr ? load_elem(bias, btype, n) : 0.f));
            }
        }
}

// ---- bias gradient: column sums of dy ----------------------------------------------------------------------------------
// A workgroup takes 32 slots of columns x 8 rows at a time over a slice of the rows; slices meet in `part` and are added in order.
template <typename T>
__global__ __launch_bounds__(256) void k_mx4_colsum(const T* __restrict__ dy, int64_t lddy, int M, int N, float* __restrict__ part) {
    constexpr int VEC = Elem<T>::VEC;
    __shared__ float s_sum[8][32][VEC];
    const int cl = threadIdx.x & 31, rl = threadIdx.x >> 5;
    const int64_t c0 = ((int64_t)blockIdx.x * 32 + cl) * VEC;
    float a[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) a[i] = 0.f;
    if (c0 < N)
        for (int64_t m = (int64_t)blockIdx.y * 8 + rl; m < M; m += (int64_t)gridDim.y * 8) {
            float v[VEC];
            load_slot(dy + m * lddy, c0, N, 0.f, v);
#pragma unroll
            for (int i = 0; i < VEC; ++i) a[i] += v[i];
        }
#pragma unroll
    for (int i = 0; i < VEC; ++i) s_sum[rl][cl][i] = a[i];
    __syncthreads();
    for (int o = threadIdx.x; o < 32 * VEC; o += 256) {
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) v += (&s_sum[k][0][0])[o];
        const int64_t c = (int64_t)blockIdx.x * 32 * VEC + o;
        if (c < N) part[(int64_t)blockIdx.y * N + c] = v;
    }
}
__global__ __launch_bounds__(256) void k_mx4_colsum_join(const float* __restrict__ part, int slices, int N, void* db, int dtype) {
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (c >= N) return;
    float v = 0.f;
    for (int k = 0; k < slices; ++k) v += part[(int64_t)k * N + c];
    store_elem(db, dtype, c, v);
}
static inline int mx4_colsum_slices(int M) { return M <= 128 ? 1 : M <= 2048 ? (M + 127) / 128 : 16; }

static inline int mx4_blocks(int K) { return K / 32 + (K % 32 != 0); }

static int mx4_check(const char* what, const void* codes, const void* scales, int64_t rows, int32_t K) {
    DRM_REQUIRE(codes && scales && aligned16(codes), DRM_EINVAL, "%s: null or misaligned codes (16 bytes) or scales", what);
    DRM_REQUIRE(rows >= 0 && K >= 1 && K <= INT_MAX - 256, DRM_EINVAL, "%s: rows=%lld K=%d", what, (long long)rows, K);
    return DRM_OK;
}
static int mx4_check_product(const char* what, const void* x, int64_t ldx, int dtype, int32_t width, const void* bias, int bias_dtype,
                             const void* y, int64_t ldy, int32_t out, int32_t M) {
    DRM_REQUIRE(x && y, DRM_EINVAL, "%s: null pointer", what);
    DRM_REQUIRE(elem_ok(dtype) && (!bias || elem_ok(bias_dtype)), DRM_ENOTSUP, "%s: element types %d / %d (fp32, bf16 or fp16)", what, dtype, bias_dtype);
    DRM_REQUIRE(M >= 1 && out >= 1 && M <= INT_MAX - 256 && out <= INT_MAX - 256 && ldx >= width && ldy >= out, DRM_EINVAL,
                "%s: M=%d N=%d, row strides %lld and %lld", what, M, out, (long long)ldx, (long long)ldy);
    return DRM_OK;
}
static int mx4_check_grid(const char* what, int M, int rows_per) {
    DRM_REQUIRE((M + rows_per - 1) / rows_per <= 65535, DRM_ENOTSUP, "%s: M=%d rows (at most %d)", what, M, 65535 * rows_per);
    return DRM_OK;
}
static inline int mx4_stream_grid(int64_t quads) { return (int)(quads < 256 * 16384ll ? (quads + 255) / 256 : 16384); }

}  // namespace drm

using namespace drm;

extern "C" int drm_mx4_quantize(const void* x, int64_t ldx, int32_t dtype, int64_t rows, int32_t K, uint8_t* codes, uint8_t* scales,
                                drm_stream_t stream) {
    if (rows == 0 && K >= 1) return DRM_OK;
    if (int rc = mx4_check(__func__, codes, scales, rows, K)) return rc;
    DRM_REQUIRE(x && ldx >= K, DRM_EINVAL, "null pointer or row stride %lld below K=%d", (long long)ldx, K);
    DRM_REQUIRE(elem_ok(dtype), DRM_ENOTSUP, "element type %d (fp32, bf16 or fp16)", dtype);
    hipStream_t s = (hipStream_t)stream;
    const int nb = mx4_blocks(K);
    ProfScope ps(PC_ELEMENTWISE, s, 4.0 * rows * K, (double)rows * K * elem_bytes(dtype) + (double)rows * nb * 17);
    return with_elem(dtype, [&](auto tag) -> int {
        using T = decltype(tag);
        k_mx4_quantize<T><<<mx4_stream_grid(rows * nb * 4), 256, 0, s>>>((const T*)x, ldx, rows, K, nb, codes, scales);
        DRM_LAUNCH_CHECK();
        return DRM_OK;
    });
}

extern "C" int drm_mx4_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t rows, int32_t K, void* y, int64_t ldy,
                                  int32_t dtype, drm_stream_t stream) {
    if (rows == 0 && K >= 1) return DRM_OK;
    if (int rc = mx4_check(__func__, codes, scales, rows, K)) return rc;
    DRM_REQUIRE(y && ldy >= K, DRM_EINVAL, "null pointer or row stride %lld below K=%d", (long long)ldy, K);
    DRM_REQUIRE(elem_ok(dtype), DRM_ENOTSUP, "element type %d (fp32, bf16 or fp16)", dtype);
    hipStream_t s = (hipStream_t)stream;
    const int nb = mx4_blocks(K);
    ProfScope ps(PC_ELEMENTWISE, s, 2.0 * rows * K, (double)rows * K * elem_bytes(dtype) + (double)rows * nb * 17);
    return with_elem(dtype, [&](auto tag) -> int {
        using T = decltype(tag);
        k_mx4_dequantize<T><<<mx4_stream_grid(rows * nb * 4), 256, 0, s>>>(codes, scales, rows, K, nb, (T*)y, ldy);
        DRM_LAUNCH_CHECK();
        return DRM_OK;
    });
}

extern "C" int drm_mx4_linear(const void* x, int64_t ldx, int32_t dtype, const uint8_t* codes, const uint8_t* scales, const void* bias,
                              int32_t bias_dtype, void* y, int64_t ldy, int32_t M, int32_t N, int32_t K, drm_stream_t stream) {
    if (M == 0 && N >= 1 && K >= 1) return DRM_OK;
    if (int rc = mx4_check(__func__, codes, scales, N, K)) return rc;
    if (int rc = mx4_check_product(__func__, x, ldx, dtype, K, bias, bias_dtype, y, ldy, N, M)) return rc;
    if (int rc = mx4_check_grid(__func__, M, 128)) return rc;
    hipStream_t s = (hipStream_t)stream;
    const Mx4 W{codes, scales, N, mx4_blocks(K)};
    ProfScope ps(M <= 64 ? PC_LINEAR : PC_LINEAR_BIG, s, 2.0 * M * N * K, ((double)M * K + (double)M * N) * elem_bytes(dtype) + (double)N * W.nb * 17);
    return with_elem(dtype, [&](auto tag) -> int {
        using T = decltype(tag);
        const int grid = (N + 15) / 16;
        if (M <= 16) k_mx4_rows<T, 1, 8><<<grid, 512, 0, s>>>((const T*)x, ldx, W, bias, bias_dtype, (T*)y, ldy, M, K);
        else if (M <= 32) k_mx4_rows<T, 2, 8><<<grid, 512, 0, s>>>((const T*)x, ldx, W, bias, bias_dtype, (T*)y, ldy, M, K);
        else if (M <= 64) k_mx4_rows<T, 4, 8><<<grid, 512, 0, s>>>((const T*)x, ldx, W, bias, bias_dtype, (T*)y, ldy, M, K);
        else k_mx4_tile<T, false><<<dim3((N + 127) / 128, (M + 127) / 128), 256, 0, s>>>((const T*)x, ldx, W, bias, bias_dtype, (T*)y, ldy, M, N, K);
        DRM_LAUNCH_CHECK();
        return DRM_OK;
    });
}

extern "C" int drm_mx4_linear_dgrad(const void* dy, int64_t lddy, int32_t dtype, const uint8_t* codes, const uint8_t* scales, void* dx,
                                    int64_t lddx, int32_t M, int32_t N, int32_t K, drm_stream_t stream) {
    if (M == 0 && N >= 1 && K >= 1) return DRM_OK;
    if (int rc = mx4_check(__func__, codes, scales, N, K)) return rc;
    if (int rc = mx4_check_product(__func__, dy, lddy, dtype, N, nullptr, 0, dx, lddx, K, M)) return rc;
    if (int rc = mx4_check_grid(__func__, M, 128)) return rc;
    DRM_REQUIRE(N >= 1, DRM_EINVAL, "N=%d", N);
    hipStream_t s = (hipStream_t)stream;
    const Mx4 W{codes, scales, N, mx4_blocks(K)};
    ProfScope ps(PC_LINEAR_BIG, s, 2.0 * M * N * K, ((double)M * K + (double)M * N) * elem_bytes(dtype) + (double)N * W.nb * 17);
    return with_elem(dtype, [&](auto tag) -> int {
        using T = decltype(tag);
        k_mx4_tile<T, true><<<dim3((K + 127) / 128, (M + 127) / 128), 256, 0, s>>>((const T*)dy, lddy, W, nullptr, 0, (T*)dx, lddx, M, K, N);
        DRM_LAUNCH_CHECK();
        return DRM_OK;
    });
}

extern "C" int drm_mx4_product(const uint8_t* x_codes, const uint8_t* x_scales, const uint8_t* w_codes, const uint8_t* w_scales,
                               const void* bias, int32_t bias_dtype, void* y, int64_t ldy, int32_t y_dtype, int32_t M, int32_t N,
                               int32_t K, drm_stream_t stream) {
    if (M == 0 && N >= 1 && K >= 1) return DRM_OK;
    if (int rc = mx4_check(__func__, x_codes, x_scales, M, K)) return rc;
    if (int rc = mx4_check(__func__, w_codes, w_scales, N, K)) return rc;
    if (int rc = mx4_check_product(__func__, x_codes, K, y_dtype, K, bias, bias_dtype, y, ldy, N, M)) return rc;
    if (int rc = mx4_check_grid(__func__, M, 64)) return rc;
    hipStream_t s = (hipStream_t)stream;
    const Mx4 X{x_codes, x_scales, M, mx4_blocks(K)}, W{w_codes, w_scales, N, mx4_blocks(K)};
    ProfScope ps(PC_LINEAR_BIG, s, 2.0 * M * N * K, (double)M * N * elem_bytes(y_dtype) + ((double)M + N) * W.nb * 17);
    return with_elem(y_dtype, [&](auto tag) -> int {
        using T = decltype(tag);
        k_mx4_product<T><<<dim3((N + 63) / 64, (M + 63) / 64), 256, 0, s>>>(X, W, bias, bias_dtype, (T*)y, ldy);
        DRM_LAUNCH_CHECK();
        return DRM_OK;
    });
}

extern "C" size_t drm_mx4_bias_grad_workspace_bytes(int32_t M, int32_t N) {
    if (M < 1 || N < 1) return 0;
    return (size_t)mx4_colsum_slices(M) * N * sizeof(float);
}

extern "C" int drm_mx4_bias_grad(const void* dy, int64_t lddy, int32_t dtype, void* db, int32_t db_dtype, int32_t M, int32_t N,
                                 void* workspace, size_t workspace_bytes, drm_stream_t stream) {
    DRM_REQUIRE(dy && db, DRM_EINVAL, "null pointer");
    DRM_REQUIRE(elem_ok(dtype) && elem_ok(db_dtype), DRM_ENOTSUP, "element types %d / %d (fp32, bf16 or fp16)", dtype, db_dtype);
    DRM_REQUIRE(M >= 1 && N >= 1 && N <= INT_MAX - 512 && lddy >= N, DRM_EINVAL, "M=%d N=%d row stride %lld", M, N, (long long)lddy);
    const size_t need = drm_mx4_bias_grad_workspace_bytes(M, N);
    DRM_REQUIRE(workspace && workspace_bytes >= need, DRM_EINVAL, "workspace of %zu bytes, %zu needed", workspace ? workspace_bytes : (size_t)0, need);
    hipStream_t s = (hipStream_t)stream;
    const int slices = mx4_colsum_slices(M);
    ProfScope ps(PC_ELEMENTWISE, s, (double)M * N, (double)M * N * elem_bytes(dtype));
    const int rc = with_elem(dtype, [&](auto tag) -> int {
        using T = decltype(tag);
        constexpr int COLS = 32 * Elem<T>::VEC;
        k_mx4_colsum<T><<<dim3((N + COLS - 1) / COLS, slices), 256, 0, s>>>((const T*)dy, lddy, M, N, (float*)workspace);
        DRM_LAUNCH_CHECK();
        return DRM_OK;
    });
    if (rc != DRM_OK) return rc;
    k_mx4_colsum_join<<<(N + 255) / 256, 256, 0, s>>>((const float*)workspace, slices, N, db, db_dtype);
    DRM_LAUNCH_CHECK();
    return DRM_OK;
}
