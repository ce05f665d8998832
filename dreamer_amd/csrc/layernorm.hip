// LayerNorm over the rows of a matrix, forward and backward with the reduction of the weight's and the bias's gradient.
//
//   m = mean(x), r = 1 / sqrt(mean((x - m)^2) + eps), xh = (x - m) r, y = xh w + b
//   dx = r (g - mean(g) - xh mean(g xh)),  g = dy w;      dw = sum over rows of dy xh;      db = sum over rows of dy
//
// Both directions are streams: forward reads x and writes y, backward reads x and dy and writes dx, and that is what bounds them.
// A row is held in registers between its statistics and its results (eight lanes to one wave for short rows, else one
// workgroup), so that x is read once and the variance is taken about the mean.  Workgroups walk over rows: the weight and the
// bias stay in registers for all of them, and so do the column sums of the backward pass, which go to `partials` once per
// workgroup and are added there in a fixed order (no atomics: results do not depend on the order in which workgroups run).
// Rates of the bytes that must move, where a copy of 4 GiB reaches 4.7 TB/s (smaller ones stay in part in the caches):
//   bf16 16384 x 4096  forward 45 us (5.9 TB/s), backward 80 us (5.0);   1048576 x 64  48 us (5.6), 82 us (4.9)
//   fp32 65536 x 512   forward 41 us (6.5),      backward 83 us (4.9);   4096 x 16384  98 us (5.5), 168 us (4.8)
// (recorded graph of twenty calls in a row, per call, as all times in this file; by itself under the profiler a kernel of this size
// takes up to a tenth more or less: bf16 16384 x 4096 forward 43 us, 4096 x 16384 forward 50 us in a row and 56 us by itself)
#include "colsum.hpp"

#include <algorithm>
#include <type_traits>

namespace drm {

// sums of two values over the TPB threads that share a row; every thread receives them.  `buf` alternates between calls so
// that one barrier per call is enough.
template <int TPB>
__device__ __forceinline__ void row_sum2(float& a, float& b, float (*buf)[2]) {
    constexpr int G = TPB < 64 ? TPB : 64;
    a = group_sum<G>(a);
    b = group_sum<G>(b);
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

// What a thread holds of a row: CH slots as they lie in memory, TPB threads per row.  All loads of a row are issued together, and
// those of the next row before this one is worked on.  Each pass over the part converts anew (`renew` keeps the compiler from
// holding the fp32 values from one pass to the next: at two bytes an element they would take twice the registers).
template <typename T, int TPB, int CH>
struct RowPart {
    static constexpr int VEC = Elem<T>::VEC;
    Slot<T> s[CH];
    __device__ __forceinline__ void load(const T* __restrict__ row, int t, int E) {
#pragma unroll
        for (int c = 0; c < CH; ++c) s[c] = raw_slot(row, (c * TPB + t) * VEC, E);
    }
    __device__ __forceinline__ void renew() {
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                u32x4 r = __builtin_bit_cast(u32x4, s[c]);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    uint32_t d = r[k];
                    asm volatile("" : "+v"(d));
                    r[k] = d;
                }
                s[c] = __builtin_bit_cast(Slot<T>, r);
            }
        }
    }
    // f(value, c, i) for every element; one that is not its slot's own (see raw_slot) comes as `fill`
    template <typename F>
    __device__ __forceinline__ void each_of(int c, int t, int E, float fill, F&& f) const {
        const int at = (c * TPB + t) * VEC, foreign = at - (int)slot_at<T>(at, E);
#pragma unroll
        for (int i = 0; i < VEC; ++i) f(i >= foreign ? (float)s[c].v[i] : fill, c, i);
    }
    template <typename F>
    __device__ __forceinline__ void each(int t, int E, float fill, F&& f) const {
#pragma unroll
        for (int c = 0; c < CH; ++c) each_of(c, t, E, fill, f);
    }
    // store f(value, c, i); a slot that was moved back writes some of its neighbour's results once more, computed like the others
    template <typename F>
    __device__ __forceinline__ void store(T* __restrict__ row, int t, int E, F&& f) const {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int at = (c * TPB + t) * VEC;
            Slot<T> o;
#pragma unroll
            for (int i = 0; i < VEC; ++i) o.v[i] = (T)f((float)s[c].v[i], c, i);
            if (at < E) *reinterpret_cast<Slot<T>*>(row + slot_at<T>(at, E)) = o;
        }
    }
};

// w, b (fp32 or the rows' type) at the positions of a thread's slots; all loads under way together
template <typename T, int TPB, int CH>
__device__ __forceinline__ void load_columns(const void* p, int type, float absent, int t, int E, float (&v)[CH][Elem<T>::VEC]) {
    constexpr int VEC = Elem<T>::VEC;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[c][i] = absent;
    if (p == nullptr) return;
    if (type == DRM_F32) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const float* at = reinterpret_cast<const float*>(p) + slot_at<T>((c * TPB + t) * VEC, E);
#pragma unroll
            for (int h = 0; h < VEC; h += 4) {
                const Slot<float> s = *reinterpret_cast<const Slot<float>*>(at + h);
#pragma unroll
                for (int i = 0; i < 4; ++i) v[c][h + i] = s.v[i];
            }
        }
    } else {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const Slot<T> s = raw_slot(reinterpret_cast<const T*>(p), (c * TPB + t) * VEC, E);
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[c][i] = (float)s.v[i];
        }
    }
}

// the same for one slot: whole ones by wide loads
template <typename T>
__device__ __forceinline__ void load_column(const void* p, int type, float absent, int64_t e, int E, float (&v)[Elem<T>::VEC]) {
    constexpr int VEC = Elem<T>::VEC;
    if (p == nullptr || e + VEC > E) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = p != nullptr ? load_elem(p, type, min(e + i, (int64_t)E - 1)) : absent;
    } else if (type == DRM_F32) {
#pragma unroll
        for (int h = 0; h < VEC; h += 4) {
            const Slot<float> s = *reinterpret_cast<const Slot<float>*>(reinterpret_cast<const float*>(p) + e + h);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[h + i] = s.v[i];
        }
    } else {
        const Slot<T> s = *reinterpret_cast<const Slot<T>*>(reinterpret_cast<const T*>(p) + e);
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = (float)s.v[i];
    }
}

// TPB threads per row: up to 64 one or several rows per wave (256 threads a workgroup), above one workgroup per row.
// KEEP: the weight and the bias stay in registers from row to row; without, they are read again (rows of more than 16 elements
// a thread)
template <typename T, int TPB, int CH, bool KEEP>
__global__ __launch_bounds__(TPB <= 64 ? 256 : TPB) void k_norm_fwd(const T* __restrict__ x, int64_t ldx, const void* w, const void* b,
                                                                    int wtype, T* __restrict__ y, int64_t ldy,
                                                                    float* __restrict__ mean, float* __restrict__ rstd, int64_t N,
                                                                    int E, float eps) {
    constexpr int VEC = Elem<T>::VEC, RPB = TPB <= 64 ? 256 / TPB : 1;
    using Part = RowPart<T, TPB, CH>;
    __shared__ float s_buf[2][TPB <= 64 ? 1 : TPB / 64][2];
    const int t = threadIdx.x % TPB;
    float wv[CH][VEC], bv[CH][VEC];
    if constexpr (KEEP) {
        load_columns<T, TPB, CH>(w, wtype, 1.f, t, E, wv);
        load_columns<T, TPB, CH>(b, wtype, 0.f, t, E, bv);
    }
    const float inv = 1.f / (float)E;
    const int64_t step = (int64_t)gridDim.x * RPB;
    Part next;
    int64_t n = (int64_t)blockIdx.x * RPB + threadIdx.x / TPB;
    next.load(x + min(n, N - 1) * ldx, t, E);
    // (uniform trip count: groups of a workgroup whose rows have run out go on with the last row and store nothing)
    for (int64_t base = (int64_t)blockIdx.x * RPB; base < N; base += step, n += step) {
        Part part = next;
        next.load(x + min(n + step, N - 1) * ldx, t, E);
        float sum = 0.f, q = 0.f;
        part.each(t, E, 0.f, [&](float v, int, int) { sum += v; });
        const float m = row_sum<TPB>(sum, s_buf[0]) * inv;
        part.renew();
        part.each(t, E, m, [&](float v, int, int) { q = fmaf(v - m, v - m, q); });
        const float r = 1.f / sqrtf(row_sum<TPB>(q, s_buf[1]) * inv + eps);
        if (n >= N) continue;
        if (t == 0 && mean != nullptr) { mean[n] = m; rstd[n] = r; }
        if constexpr (!KEEP) {
            load_columns<T, TPB, CH>(w, wtype, 1.f, t, E, wv);
            load_columns<T, TPB, CH>(b, wtype, 0.f, t, E, bv);
        }
        part.renew();
        part.store(y + n * ldy, t, E, [&](float v, int c, int i) { return fmaf((v - m) * r, wv[c][i], bv[c][i]); });
    }
}

// Rows shorter than a slot: a row per thread, its elements one by one (a wave's rows lie side by side, so that their lines are
// read once).  2000000 x 3 fp32: 12 us forward, 22 us backward; with a workgroup per row 1.2 and 25 ms.
template <typename T>
__global__ __launch_bounds__(256) void k_norm_fwd_narrow(const T* __restrict__ x, int64_t ldx, const void* w, const void* b, int wtype,
                                                         T* __restrict__ y, int64_t ldy, float* __restrict__ mean,
                                                         float* __restrict__ rstd, int64_t N, int E, float eps) {
    constexpr int M = Elem<T>::VEC - 1;
    const float inv = 1.f / (float)E;
    float wv[M], bv[M], v[M];
#pragma unroll
    for (int i = 0; i < M; ++i) {
        wv[i] = i < E && w != nullptr ? load_elem(w, wtype, i) : 1.f;
        bv[i] = i < E && b != nullptr ? load_elem(b, wtype, i) : 0.f;
    }
    for (int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x; n < N; n += (int64_t)gridDim.x * 256) {
        float sum = 0.f, q = 0.f;
#pragma unroll
        for (int i = 0; i < M; ++i) { v[i] = i < E ? (float)x[n * ldx + i] : 0.f; sum += v[i]; }
        const float m = sum * inv;
#pragma unroll
        for (int i = 0; i < M; ++i) q += i < E ? (v[i] - m) * (v[i] - m) : 0.f;
        const float r = 1.f / sqrtf(q * inv + eps);
        if (mean != nullptr) { mean[n] = m; rstd[n] = r; }
#pragma unroll
        for (int i = 0; i < M; ++i)
            if (i < E) y[n * ldy + i] = (T)fmaf((v[i] - m) * r, wv[i], bv[i]);
    }
}
// backward: a workgroup's column sums by lanes, then wave after wave (see k_norm_bwd for `partials`)
template <typename T>
__global__ __launch_bounds__(256) void k_norm_bwd_narrow(const T* __restrict__ x, int64_t ldx, const T* __restrict__ dy, int64_t lddy,
                                                         const void* w, int wtype, const float* __restrict__ mean,
                                                         const float* __restrict__ rstd, T* __restrict__ dx,
                                                         float* __restrict__ partials, int64_t N, int E) {
    constexpr int M = Elem<T>::VEC - 1;
    __shared__ float s_wave[4][2 * M];
    const float inv = 1.f / (float)E;
    float wv[M], aw[M], ab[M], d[M], h[M];
#pragma unroll
    for (int i = 0; i < M; ++i) {
        wv[i] = i < E && w != nullptr ? load_elem(w, wtype, i) : 1.f;
        aw[i] = 0.f;
        ab[i] = 0.f;
    }
    for (int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x; n < N; n += (int64_t)gridDim.x * 256) {
        const float m = mean[n], r = rstd[n];
        float s = 0.f, q = 0.f;
#pragma unroll
        for (int i = 0; i < M; ++i) {
            d[i] = i < E ? (float)dy[n * lddy + i] : 0.f;
            h[i] = i < E ? ((float)x[n * ldx + i] - m) * r : 0.f;
            aw[i] = fmaf(d[i], h[i], aw[i]);
            ab[i] += d[i];
            s = fmaf(d[i], wv[i], s);
            q = fmaf(d[i] * wv[i], h[i], q);
        }
        if (dx == nullptr) continue;
        s *= inv; q *= inv;
#pragma unroll
        for (int i = 0; i < M; ++i)
            if (i < E) dx[n * (int64_t)E + i] = (T)(r * (fmaf(d[i], wv[i], -s) - h[i] * q));
    }
    if (partials == nullptr) return;
#pragma unroll
    for (int i = 0; i < M; ++i) {
        aw[i] = group_sum<64>(aw[i]);
        ab[i] = group_sum<64>(ab[i]);
    }
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
        for (int i = 0; i < M; ++i) { s_wave[threadIdx.x >> 6][i] = aw[i]; s_wave[threadIdx.x >> 6][M + i] = ab[i]; }
    }
    __syncthreads();
    const int i = threadIdx.x % M, half = threadIdx.x / M;
    if (half < 2 && i < E)
        partials[((int64_t)blockIdx.x * 2 + half) * E + i] =
            (s_wave[0][half * M + i] + s_wave[1][half * M + i]) + (s_wave[2][half * M + i] + s_wave[3][half * M + i]);
}

// Rows too long for registers: three walks over the row (the second and third find it in the caches unless it is longer than
// those).  One workgroup per row, four slots under way per thread: at 512 threads they fit the registers (1024 x 65536 bf16
// 80 us, 3.4 TB/s; at 1024 threads 110 us, spilled).
template <typename T, int TPB>
__global__ __launch_bounds__(TPB) void k_norm_fwd_long(const T* __restrict__ x, int64_t ldx, const void* w, const void* b, int wtype,
                                                       T* __restrict__ y, int64_t ldy, float* __restrict__ mean,
                                                       float* __restrict__ rstd, int64_t N, int E, float eps) {
    constexpr int VEC = Elem<T>::VEC, U = 4, STEP = TPB * VEC;
    __shared__ float s_buf[2][TPB / 64][2];
    const float inv = 1.f / (float)E;
    const int64_t bulk = (int64_t)E / (U * STEP) * (U * STEP);       // whole slots of every thread
    for (int64_t n = blockIdx.x; n < N; n += gridDim.x) {
        const T* row = x + n * ldx;
        float s = 0.f, q = 0.f;
        auto walk = [&](auto&& f) {
            for (int64_t e = (int64_t)threadIdx.x * VEC; e < bulk; e += U * STEP) {
                Slot<T> raw[U];
#pragma unroll
                for (int u = 0; u < U; ++u) raw[u] = *reinterpret_cast<const Slot<T>*>(row + e + u * STEP);
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    float v[VEC];
#pragma unroll
                    for (int i = 0; i < VEC; ++i) v[i] = (float)raw[u].v[i];
                    f(v, VEC, e + u * STEP);
                }
            }
            for (int64_t e = bulk + (int64_t)threadIdx.x * VEC; e < E; e += STEP) {
                float v[VEC];
                load_slot(row, e, E, 0.f, v);
                f(v, (int)min((int64_t)VEC, E - e), e);
            }
        };
        walk([&](const float (&v)[VEC], int, int64_t) {
            float p = 0.f;
#pragma unroll
            for (int i = 0; i < VEC; ++i) p += v[i];
            s += p;
        });
        const float m = row_sum<TPB>(s, s_buf[0]) * inv;
        walk([&](const float (&v)[VEC], int have, int64_t) {
            float p = 0.f;
#pragma unroll
            for (int i = 0; i < VEC; ++i) p += i < have ? (v[i] - m) * (v[i] - m) : 0.f;
            q += p;
        });
        const float r = 1.f / sqrtf(row_sum<TPB>(q, s_buf[1]) * inv + eps);
        if (threadIdx.x == 0 && mean != nullptr) { mean[n] = m; rstd[n] = r; }
        walk([&](const float (&v)[VEC], int, int64_t e) {
            float o[VEC], wv[VEC], bv[VEC];
            load_column<T>(w, wtype, 1.f, e, E, wv);
            load_column<T>(b, wtype, 0.f, e, E, bv);
#pragma unroll
            for (int i = 0; i < VEC; ++i) o[i] = fmaf((v[i] - m) * r, wv[i], bv[i]);
            store_slot(y + n * ldy, e, E, o);
        });
    }
}

// partials: (gridDim.x, 2, E): column sums of dy xh and of dy over the rows this workgroup walked
template <typename T, int TPB, int CH>
__global__ __launch_bounds__(TPB <= 64 ? 256 : TPB, 4) void k_norm_bwd(const T* __restrict__ x, int64_t ldx, const T* __restrict__ dy,
                                                                    int64_t lddy, const void* w, int wtype,
                                                                    const float* __restrict__ mean, const float* __restrict__ rstd,
                                                                    T* __restrict__ dx, float* __restrict__ partials, int64_t N,
                                                                    int E) {
    constexpr int VEC = Elem<T>::VEC, RPB = TPB <= 64 ? 256 / TPB : 1;
    // Sixteen elements at 1024 threads, 128 registers each: the weight is read again for every row, and the column sums stay in
    // LDS, each thread's its own (4096 x 16384 bf16: 116 us, 3.5 TB/s; all in registers, which spill, 170 us).
    constexpr bool KEEP = CH * VEC <= 8, AHEAD = KEEP || sizeof(T) == 2;      // (fp32: no registers left for the next row's)
    static_assert(KEEP || TPB > 64, "column sums in LDS: one row per workgroup");
    using Part = RowPart<T, TPB, CH>;
    __shared__ float s_buf[2][TPB <= 64 ? 1 : TPB / 64][2];
    __shared__ float s_cols[TPB <= 64 ? TPB * CH * VEC : 1];
    __shared__ f32x4 s_sums[KEEP ? 1 : CH * VEC / 4 * 2][KEEP ? 1 : TPB];
    const int t = threadIdx.x % TPB;
    float wv[CH][VEC], aw[CH][VEC], ab[CH][VEC];
    auto sums_from = [&](int c) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            aw[c][i] = s_sums[(c * VEC + i) / 4 * 2][t][i & 3];
            ab[c][i] = s_sums[(c * VEC + i) / 4 * 2 + 1][t][i & 3];
        }
    };
    auto sums_to = [&](int c) {
#pragma unroll
        for (int i = 0; i < VEC; i += 4) {
            s_sums[(c * VEC + i) / 4 * 2][t] = f32x4{aw[c][i], aw[c][i + 1], aw[c][i + 2], aw[c][i + 3]};
            s_sums[(c * VEC + i) / 4 * 2 + 1][t] = f32x4{ab[c][i], ab[c][i + 1], ab[c][i + 2], ab[c][i + 3]};
        }
    };
    if constexpr (KEEP) load_columns<T, TPB, CH>(w, wtype, 1.f, t, E, wv);
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < VEC; ++i) { aw[c][i] = 0.f; ab[c][i] = 0.f; }
    if constexpr (!KEEP) {
#pragma unroll
        for (int c = 0; c < CH; ++c) sums_to(c);
    }
    const float inv = 1.f / (float)E;
    const int64_t step = (int64_t)gridDim.x * RPB;
    Part nx, nd;
    float nm = 0.f, nr = 0.f;
    int64_t n = (int64_t)blockIdx.x * RPB + threadIdx.x / TPB;
    auto fetch = [&](int64_t at) {
        const int64_t k = min(at, N - 1);
        nx.load(x + k * ldx, t, E);
        nd.load(dy + k * lddy, t, E);
        nm = mean[k];
        nr = rstd[k];
    };
    if constexpr (AHEAD) fetch(n);
    int flip = 0;
    for (int64_t base = (int64_t)blockIdx.x * RPB; base < N; base += step, n += step, flip ^= 1) {
        if constexpr (!AHEAD) fetch(n);
        Part px = nx, pd = nd;
        const float m = nm, r = nr;
        const bool live = n < N;                                  // (a group of a wave without a row: nothing to add)
        if constexpr (AHEAD) fetch(n + step);
        if constexpr (!KEEP) load_columns<T, TPB, CH>(w, wtype, 1.f, t, E, wv);
        float s = 0.f, q = 0.f;
#pragma unroll
        for (int k = 0; k < CH; ++k) {
            if constexpr (!KEEP) sums_from(k);
            pd.each_of(k, t, E, 0.f, [&](float d, int c, int i) {
                if (TPB <= 64 && !live) d = 0.f;
                const float h = ((float)px.s[c].v[i] - m) * r, gw = d * wv[c][i];
                aw[c][i] = fmaf(d, h, aw[c][i]);
                ab[c][i] += d;
                s += gw;
                q = fmaf(gw, h, q);
            });
            if constexpr (!KEEP) sums_to(k);
        }
        row_sum2<TPB>(s, q, s_buf[flip]);
        if (dx != nullptr && live) {
            s *= inv; q *= inv;
            if constexpr (!KEEP) load_columns<T, TPB, CH>(w, wtype, 1.f, t, E, wv);
            px.renew();
            pd.renew();
            pd.store(dx + n * (int64_t)E, t, E, [&](float d, int c, int i) {
                return r * (fmaf(d, wv[c][i], -s) - ((float)px.s[c].v[i] - m) * r * q);
            });
        }
    }
    if (partials == nullptr) return;
    float* pw = partials + (int64_t)blockIdx.x * 2 * E;
    if constexpr (TPB <= 64) {
        // rows of one wave first, then the four waves one after the other
        if constexpr (TPB < 64) {
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    if constexpr (TPB <= 8) { aw[c][i] += xor_lane<8>(aw[c][i]); ab[c][i] += xor_lane<8>(ab[c][i]); }
                    if constexpr (TPB <= 16) { aw[c][i] += xor_lane<16>(aw[c][i]); ab[c][i] += xor_lane<16>(ab[c][i]); }
                    aw[c][i] += xor_lane<32>(aw[c][i]); ab[c][i] += xor_lane<32>(ab[c][i]);
                }
        }
        const int wave = threadIdx.x >> 6;
        const bool first = (threadIdx.x & 63) < TPB;
#pragma unroll
        for (int half = 0; half < 2; ++half)
            for (int k = 0; k < 4; ++k) {
                __syncthreads();
                if (wave != k || !first) continue;
#pragma unroll
                for (int c = 0; c < CH; ++c)
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        const int at = (c * TPB + t) * VEC;
                        const float sum = (k == 0 ? 0.f : s_cols[at + i]) + (half == 0 ? aw[c][i] : ab[c][i]);
                        if (k < 3) s_cols[at + i] = sum;
                        else if (at < E && owned<T>(at, E, i)) pw[(int64_t)half * E + slot_at<T>(at, E) + i] = sum;
                    }
            }
    } else {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            if constexpr (!KEEP) sums_from(c);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const int at = (c * TPB + t) * VEC;
                if (at < E && owned<T>(at, E, i)) {
                    pw[slot_at<T>(at, E) + i] = aw[c][i];
                    pw[E + slot_at<T>(at, E) + i] = ab[c][i];
                }
            }
        }
    }
}

// The long rows backward, x and dy read twice: the two row means first (2048 x 32768 bf16, all three kernels: 143 us) ...
template <typename T, int TPB>
__global__ __launch_bounds__(TPB) void k_norm_bwd_sums(const T* __restrict__ x, int64_t ldx, const T* __restrict__ dy, int64_t lddy,
                                                        const void* w, int wtype, const float* __restrict__ mean,
                                                        const float* __restrict__ rstd, float* __restrict__ sums, int64_t N, int E) {
    constexpr int VEC = Elem<T>::VEC, U = 2, STEP = TPB * VEC;
    __shared__ float s_buf[2][TPB / 64][2];
    const int64_t bulk = (int64_t)E / (U * STEP) * (U * STEP);       // whole slots of every thread
    int flip = 0;
    for (int64_t n = blockIdx.x; n < N; n += gridDim.x, flip ^= 1) {
        const float m = mean[n], r = rstd[n];
        const T *rx = x + n * ldx, *rg = dy + n * lddy;
        float xv[VEC], g[VEC], s = 0.f, q = 0.f;
        auto one = [&](int64_t e) {
            float ps = 0.f, pq = 0.f, wv[VEC];
            load_column<T>(w, wtype, 1.f, e, E, wv);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float gw = g[i] * wv[i];
                ps += gw;
                pq = fmaf(gw, (xv[i] - m) * r, pq);
            }
            s += ps; q += pq;
        };
        for (int64_t e = (int64_t)threadIdx.x * VEC; e < bulk; e += U * STEP) {
            Slot<T> sx[U], sg[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                sx[u] = *reinterpret_cast<const Slot<T>*>(rx + e + u * STEP);
                sg[u] = *reinterpret_cast<const Slot<T>*>(rg + e + u * STEP);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
#pragma unroll
                for (int i = 0; i < VEC; ++i) { xv[i] = (float)sx[u].v[i]; g[i] = (float)sg[u].v[i]; }
                one(e + u * STEP);
            }
        }
        for (int64_t e = bulk + (int64_t)threadIdx.x * VEC; e < E; e += STEP) {
            load_slot(rx, e, E, m, xv);
            load_slot(rg, e, E, 0.f, g);
            one(e);
        }
        row_sum2<TPB>(s, q, s_buf[flip]);
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
    auto one = [&](int64_t n, const float (&xv)[VEC], float (&g)[VEC]) {
        const float m = mean[n], r = rstd[n];
        const float s = sums != nullptr ? sums[2 * n] : 0.f, q = sums != nullptr ? sums[2 * n + 1] : 0.f;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const float h = (xv[i] - m) * r;
            aw[i] = fmaf(g[i], h, aw[i]);
            ab[i] += g[i];
            g[i] = r * (g[i] * wv[i] - fmaf(h, q, s));
        }
        if (dx != nullptr) store_slot(dx + n * (int64_t)E, e, E, g);
    };
    float xv[VEC], g[VEC];
    int64_t n = blockIdx.y;
    if (e + VEC <= E) {
        // whole slots: four rows under way
        constexpr int U = 4;
        for (; n + (U - 1) * (int64_t)gridDim.y < N; n += U * (int64_t)gridDim.y) {
            Slot<T> rx[U], rg[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                rx[u] = *reinterpret_cast<const Slot<T>*>(x + (n + u * (int64_t)gridDim.y) * ldx + e);
                rg[u] = *reinterpret_cast<const Slot<T>*>(dy + (n + u * (int64_t)gridDim.y) * lddy + e);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
#pragma unroll
                for (int i = 0; i < VEC; ++i) { xv[i] = (float)rx[u].v[i]; g[i] = (float)rg[u].v[i]; }
                one(n + u * (int64_t)gridDim.y, xv, g);
            }
        }
    }
    for (; n < N; n += gridDim.y) {
        load_slot(x + n * ldx, e, E, mean[n], xv);
        load_slot(dy + n * lddy, e, E, 0.f, g);
        one(n, xv, g);
    }
    if (partials != nullptr) {
        float* pw = partials + (int64_t)blockIdx.y * 2 * E;
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            if (e + i < E) { pw[e + i] = aw[i]; pw[E + e + i] = ab[i]; }
    }
}

// ---- host side -------------------------------------------------------------------------------------------------------
// Threads per row by the row's length: the fewest lanes whose slots cover it, at most 16 elements a thread forward and 8 backward
// (x, dy, the next row's, weight, two running column sums: 80 to 100 registers, four to five waves per SIMD).  Forward with 8
// instead: 65536 x 1024 bf16 47 us against 41, 8192 x 8192 51 against 46; backward with 16 spills or needs the LDS.
// Forward above 16384: two-byte rows up to 32768 stay in registers with the weight read again (2048 x 32768: 75 us, three
// walks 88), fp32 rows walk (1024 x 32768: 76 us, in registers 126).
constexpr int NORM_MAX_E = 1024 * 16;
template <typename T>
static constexpr int norm_max_fwd() { return sizeof(T) == 2 ? 2 * NORM_MAX_E : NORM_MAX_E; }
template <typename T>
static inline bool norm_narrow(int E) { return E < Elem<T>::VEC; }
// Workgroups that walk the rows backward; each leaves 2 E column sums.  At most about four waves per SIMD (65536 x 1024 bf16: 512
// workgroups 115 us, 1024 82 us, 2048 88 us; 16384 x 4096: 128 125 us, 256 80 us, 1024 96 us), and of four rows at least where
// rows are few (1024 x 1024: 256 workgroups 9 us, one per row 15 us).
static inline int norm_slices(int64_t N, int E, int x_dtype) {
    if (N < 1) return 1;
    const int vec = x_dtype == DRM_F32 ? 4 : 8;
    if (E > NORM_MAX_E) return (int)(N < 64 ? N : 64);
    if (E < vec) return (int)std::min<int64_t>((N + 255) / 256, 1024);
    const int64_t rpb = E <= 8 * vec ? 32 : E <= 16 * vec ? 16 : E <= 32 * vec ? 8 : E <= 512 ? 4 : 1, groups = (N + rpb - 1) / rpb;
    const int64_t cap = E <= 1024 ? 1024 : E <= 2048 ? 512 : 256, few = std::max<int64_t>(groups / 4, 128);
    return (int)std::min(groups, std::min(few, cap));
}

#define DRM_NORM_CASE(TPB, CH) return f(std::integral_constant<int, TPB>{}, std::integral_constant<int, CH>{})
template <typename T, bool BWD, typename F>
static int norm_variant(int E, F&& f) {
    constexpr int VEC = Elem<T>::VEC, C8 = 8 / VEC, C16 = 16 / VEC;
    if (E <= 8 * VEC) DRM_NORM_CASE(8, 1);
    if (E <= 16 * VEC) DRM_NORM_CASE(16, 1);
    if (E <= 32 * VEC) DRM_NORM_CASE(32, 1);
    if (E <= 64 * VEC) DRM_NORM_CASE(64, 1);
    if (E <= 512) DRM_NORM_CASE(64, C8);
    if constexpr (BWD) {
        if (E <= 1024) DRM_NORM_CASE(128, C8);
        if (E <= 2048) DRM_NORM_CASE(256, C8);
        if (E <= 4096) DRM_NORM_CASE(512, C8);
        if (E <= 8192) DRM_NORM_CASE(1024, C8);
    } else {
        if (E <= 1024) DRM_NORM_CASE(64, C16);
        if (E <= 2048) DRM_NORM_CASE(256, C8);
        if (E <= 4096) DRM_NORM_CASE(256, C16);
        if (E <= 8192) DRM_NORM_CASE(512, C16);
    }
    DRM_NORM_CASE(1024, C16);
}
#undef DRM_NORM_CASE

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
        if (norm_narrow<T>(E)) {
            k_norm_fwd_narrow<T><<<(int)std::min<int64_t>((N + 255) / 256, 2048), 256, 0, s>>>((const T*)x, ldx, w, b, w_dtype, (T*)y, ldy, mean, rstd, N, E, eps);
        } else if (E > norm_max_fwd<T>()) {
            k_norm_fwd_long<T, 512><<<(int)(N < 4096 ? N : 4096), 512, 0, s>>>((const T*)x, ldx, w, b, w_dtype, (T*)y, ldy, mean, rstd, N, E, eps);
        } else if (E > NORM_MAX_E) {
            if constexpr (sizeof(T) == 2)
                k_norm_fwd<T, 1024, 4, false><<<(int)(N < 512 ? N : 512), 1024, 0, s>>>((const T*)x, ldx, w, b, w_dtype, (T*)y, ldy, mean, rstd, N, E, eps);
        } else {
            norm_variant<T, false>(E, [&](auto tpb, auto ch) {
                constexpr int TPB = decltype(tpb)::value, CH = decltype(ch)::value, RPB = TPB <= 64 ? 256 / TPB : 1;
                // four times the workgroups that the chip holds at once (16384 x 4096 bf16 side by side 42 us, once 46, sixteen times 48);
                // of 1024 threads as many as it holds (4096 x 16384: 50 us, four times 64 us)
                const int64_t groups = (N + RPB - 1) / RPB, cap = TPB <= 64 ? 8192 : 256 * (TPB < 1024 ? 8192 : 2048) / TPB;
                k_norm_fwd<T, TPB, CH, true><<<(int)(groups < cap ? groups : cap), TPB <= 64 ? 256 : TPB, 0, s>>>((const T*)x, ldx, w, b, w_dtype, (T*)y, ldy, mean, rstd, N, E, eps);
                return 0;
            });
        }
        DRM_LAUNCH_CHECK();
        return DRM_OK;
    });
}

// (the larger of what the row types need)
extern "C" size_t drm_layer_norm_workspace_bytes(int64_t N, int32_t E) {
    if (N < 0 || E < 1) return 0;
    size_t need = 0;
    for (int t : {DRM_F32, DRM_BF16}) {
        const size_t sums = E > NORM_MAX_E ? (size_t)N * 2 * sizeof(float) : 0;
        need = std::max(need, sums + (size_t)norm_slices(N, E, t) * 2 * E * sizeof(float));
    }
    return need;
}

extern "C" int drm_layer_norm_backward(const void* x, int64_t ldx, const void* dy, int64_t lddy, int32_t x_dtype, const void* w,
                                       int32_t w_dtype, const float* mean, const float* rstd, void* dx, void* dw, void* db,
                                       int64_t N, int32_t E, void* workspace, size_t workspace_bytes, drm_stream_t stream) {
    hipStream_t s = (hipStream_t)stream;
    const bool cols = dw != nullptr || db != nullptr;
    DRM_REQUIRE(N >= 0 && E >= 1, DRM_EINVAL, "N=%lld E=%d", (long long)N, E);
    DRM_REQUIRE(elem_ok(x_dtype) && (w_dtype == DRM_F32 || w_dtype == x_dtype), DRM_ENOTSUP, "element types %d / %d", x_dtype, w_dtype);
    if (N == 0) {
        if (cols) { join_columns(nullptr, 0, 2 * (int64_t)E, E, w_dtype, dw, db, s); DRM_LAUNCH_CHECK(); }
        return DRM_OK;
    }
    if (int rc = norm_check(__func__, x, ldx, x_dtype, w_dtype, N, E)) return rc;
    DRM_REQUIRE(dy && lddy >= E && mean && rstd, DRM_EINVAL, "null pointer or row stride %lld below E=%d", (long long)lddy, E);
    if (!dx && !cols) return DRM_OK;
    DRM_REQUIRE(workspace && workspace_bytes >= drm_layer_norm_workspace_bytes(N, E), DRM_EINVAL, "workspace of %zu bytes, %zu needed",
                workspace ? workspace_bytes : (size_t)0, drm_layer_norm_workspace_bytes(N, E));
    const int slices = norm_slices(N, E, x_dtype);
    const bool walk = E > NORM_MAX_E;
    const double n = (double)N * E;
    ProfScope ps(PC_ELEMENTWISE, s, 17 * n, 3 * n * elem_bytes(x_dtype));
    float* sums = (float*)workspace;
    float* part = !cols ? nullptr : walk ? sums + 2 * N : sums;
    const int rc = with_elem(x_dtype, [&](auto tag) -> int {
        using T = decltype(tag);
        if (norm_narrow<T>(E)) {
            k_norm_bwd_narrow<T><<<slices, 256, 0, s>>>((const T*)x, ldx, (const T*)dy, lddy, w, w_dtype, mean, rstd, (T*)dx, part, N, E);
        } else if (walk) {
            if (dx != nullptr) {
                k_norm_bwd_sums<T, 1024><<<(int)(N < 4096 ? N : 4096), 1024, 0, s>>>((const T*)x, ldx, (const T*)dy, lddy, w, w_dtype, mean, rstd, sums, N, E);
                DRM_LAUNCH_CHECK();
            }
            constexpr int STRIP = 256 * Elem<T>::VEC;
            k_norm_bwd_cols<T><<<dim3((unsigned)(((int64_t)E + STRIP - 1) / STRIP), slices), 256, 0, s>>>((const T*)x, ldx, (const T*)dy, lddy, w, w_dtype, mean, rstd,
                                                                                      dx != nullptr ? sums : nullptr, (T*)dx, part, N, E);
        } else {
            norm_variant<T, true>(E, [&](auto tpb, auto ch) {
                constexpr int TPB = decltype(tpb)::value, CH = decltype(ch)::value;
                k_norm_bwd<T, TPB, CH><<<slices, TPB <= 64 ? 256 : TPB, 0, s>>>((const T*)x, ldx, (const T*)dy, lddy, w, w_dtype, mean, rstd, (T*)dx, part, N, E);
                return 0;
            });
        }
        DRM_LAUNCH_CHECK();
        return DRM_OK;
    });
    if (rc != DRM_OK || !cols) return rc;
    join_columns(part, slices, 2 * (int64_t)E, E, w_dtype, dw, db, s);
    DRM_LAUNCH_CHECK();
    return DRM_OK;
}
