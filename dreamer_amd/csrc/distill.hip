// Distillation loss from a teacher's top logits: forward and gradient over rows of V student logits.
//
// s: student logits, T: temperature, q = softmax(s / T) over the row.  The teacher is a list of (value t_j, index i_j);
// entries whose index lies outside [0, V) are absent, a row with none left has loss 0 and gradient 0.
//   without the teacher's log-sum-exp:  p_j = softmax of t_j / T over the listed entries, nothing is left over
//   with it (L, of t / T over the teacher's whole row):  p_j = exp(t_j / T - L), the rest P = max(0, 1 - sum_j p_j) is
//   compared with the student's rest Q = sum of q over the unlisted entries (P is dropped where no unlisted entry is left)
//   loss = sum_j p_j (log p_j - log q_{i_j}) + P (log P - log Q)
//   d loss / d s_v = (1 / T) (q_v (sum_j p_j + P) - sum_{j: i_j = v} p_j - [v unlisted] q_v P / Q)
//
// The rows are streams (read once forward; read once and written once backward), the list is a few hundred bytes beside
// them.  Forward keeps a running maximum and sum per thread over groups of slots (one rescaling per group), backward is one
// multiplication of exp((s - m) / T) by a factor per row.  With the teacher's log-sum-exp the unlisted entries are summed by
// themselves (a bitmap of the listed ones in LDS): log Q = -log1p(listed / unlisted) keeps its digits where Q is close to 1,
// and so does log P = log1p(-sum p).  The per-row scalars are formed in 64 bits because they are small differences of numbers
// close to 1.  Held in 32 bits, each for half a step or a few of a sum of positive terms (the loss is off by 6e-8 at 240 x 255):
// a thread's sum of exponentials (its terms come from a 32-bit exponential); the sums of a segment on their way to the join (a row
// of one segment keeps its 64 bits across threads); 1 / T as the exponent's factor, see exp_scaled; and p, which backward
// subtracts from a 32-bit q.
//
// A row is cut into segments, one workgroup each: with one segment the row is finished in the same launch, else a second kernel
// joins the segments' (maximum, sum).
// 4096 x 32768 bf16, 64 listed: forward 51 us (5.3 TB/s), with the rest 59 us (the masks; the exponentials of a row take
// half of its time), backward 95 us (5.7 TB/s).  Rows of a few thousand logits are bound by the end of a row: two logarithms and
// up to three exponentials in 64 bits, about 1.5 us of a SIMD because a wave ends one row and its lanes form the same scalars
// (65536 x 1024: 89 us, with the rest 140 us, 1.7 and 1.1 TB/s, where the bytes alone would take 32 us).
// Times here and below: recorded graph of twenty calls in a row, per call.
#include "elem.hpp"

#include <algorithm>
#include <climits>
#include <cmath>

namespace drm {

constexpr int DISTILL_SEG = 32768;     // entries a workgroup takes forward (a bitmap of 4 KiB): 4096 x 32768 with the rest 59 us (16384: 65, 8192: 70), 16 x 131072 15 us (13, 11)
constexpr int DISTILL_SEG_BWD = 4096;  // and backward, where nothing has to be joined: 4096 x 32768 bf16 95 us (16384: 113, 32768: 120), 16 x 32768 3.4 us (5.5, 8.2)
constexpr int DISTILL_MAX_K = 1024;

struct DistillRow {                    // what backward needs of a row (both factors 0: no gradient)
    float m, inside;                   // listed entries: exp((s - m) / T) * inside - p
    float m_out, outside;              // unlisted entries: exp((s - m_out) / T) * outside
};

struct DistillArgs {
    const void* s; int64_t lds; int V;
    const float* val; int64_t ldv; const int64_t* idx; int64_t ldi; int k;
    const float* lse;                  // teacher's log-sum-exp per row or nullptr
    double inv_t, inv_ts;              // 1 / T, as the teacher's and as the student's side take it
    int segs;
    float4* part;                      // (rows, segs): maximum m and sum of exp((s - m) / T) of the unlisted, of the listed entries
    float* loss; float* p; DistillRow* row;
    template <typename T> DistillArgs from(int64_t r) const {      // the rows from r on
        DistillArgs a = *this;
        a.s = (const T*)s + r * lds; a.val += r * ldv; a.idx += r * ldi; a.loss += r; a.p += r * k; a.row += r;
        if (lse != nullptr) a.lse += r;
        if (part != nullptr) a.part += r * segs;
        return a;
    }
};

// exp(d / T) for d <= 0 as 2^(d c), c = log2(e) / T rounded to 32 bits.  The per-row scalars take c ln(2) in 64 bits as the
// student's 1 / T, so that the rounding of c shifts the temperature by 2^-25 instead of making sums and logarithms disagree.
__device__ __forceinline__ float exp_scaled(float d, float c) { return __builtin_amdgcn_exp2f(d * c); }

// ---- the listed entries of a segment as a bitmap ------------------------------------------------------------------------
// true if an entry of the segment is listed more than once (valid behind the function's barrier)
__device__ __forceinline__ bool segment_bitmap(const int64_t* __restrict__ idx, int k, int v0, int v1, uint32_t* bits, int* twice) {
    for (int w = threadIdx.x; w < (v1 - v0 + 31) / 32; w += blockDim.x) bits[w] = 0;
    if (threadIdx.x == 0) *twice = 0;
    __syncthreads();
    for (int j = threadIdx.x; j < k; j += blockDim.x) {
        const int64_t i = idx[j];
        if (i < v0 || i >= v1) continue;
        const uint32_t bit = 1u << ((i - v0) & 31);
        if (atomicOr(&bits[(i - v0) >> 5], bit) & bit) *twice = 1;
    }
    __syncthreads();
    return *twice != 0;
}

// (maximum, sum of exp((s - maximum) / T)) of two sets of entries
struct MaxSum { float m; double z; };
__device__ __forceinline__ MaxSum join(MaxSum a, MaxSum b, double inv_t) {
    const float n = fmaxf(a.m, b.m);
    if (n == -INFINITY) return {n, a.z + b.z};             // nothing finite on either side
    return {n, (a.m == -INFINITY ? a.z : a.z * exp(((double)a.m - (double)n) * inv_t))
                   + (b.m == -INFINITY ? b.z : b.z * exp(((double)b.m - (double)n) * inv_t))};
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);
    return v;
}
__device__ __forceinline__ MaxSum wave_join(MaxSum a, double inv_t) {
    const float top = group_max<64>(a.m);
    const double z = a.m == -INFINITY || top == a.m ? a.z : a.z * exp(((double)a.m - (double)top) * inv_t);
    return {top, wave_sum(z)};
}

// ---- end of a row, by one wave ------------------------------------------------------------------------------------------
// `out`: the row's unlisted entries, `in` its listed ones (with the teacher's log-sum-exp); `out` all entries (without)
template <typename T>
__device__ void finish_row(const DistillArgs& A, int64_t r, MaxSum out, MaxSum in) {
    const int lane = threadIdx.x & 63;
    const T* s = (const T*)A.s + r * A.lds;
    const float* val = A.val + r * A.ldv;
    const int64_t* idx = A.idx + r * A.ldi;
    const bool with_rest = A.lse != nullptr;
    const MaxSum all = with_rest ? join(out, in, A.inv_ts) : out;
    const double logz = log(all.z);
    // the teacher's side; a list of nothing but -inf has no softmax and counts as empty
    float tmax = -INFINITY;
    int some = 0;
    for (int j = lane; j < A.k; j += 64) {
        const int64_t i = idx[j];
        if (i < 0 || i >= A.V) continue;
        tmax = fmaxf(tmax, val[j]);
        some |= with_rest || val[j] != -INFINITY;
    }
    tmax = group_max<64>(tmax);
    const bool any = __any(some);
    const double base = with_rest ? (double)A.lse[r] : (double)tmax * A.inv_t;
    double psum = 0.0;
    for (int j = lane; j < A.k; j += 64) {
        const int64_t i = idx[j];
        if (i >= 0 && i < A.V) psum += exp((double)val[j] * A.inv_t - base);
    }
    psum = wave_sum(psum);
    const double norm = with_rest ? 1.0 : 1.0 / psum, lnorm = with_rest ? 0.0 : log(psum);
    double loss = 0.0;
    for (int j = lane; j < A.k; j += 64) {
        const int64_t i = idx[j];
        float keep = 0.f;
        if (i >= 0 && i < A.V) {
            const double lp = (double)val[j] * A.inv_t - base, p = exp(lp) * norm;
            if (!(p <= 0.0)) loss += p * (lp - lnorm - (((double)(float)s[i] - (double)all.m) * A.inv_ts - logz));
            keep = (float)p;
        }
        A.p[r * A.k + j] = keep;
    }
    loss = wave_sum(loss);
    if (lane != 0) return;
    const double mass = with_rest ? psum : 1.0;
    const double rest = with_rest && out.z > 0.0 && mass < 1.0 ? 1.0 - mass : 0.0;
    DistillRow o{0.f, 0.f, 0.f, 0.f};
    if (any) {
        if (rest > 0.0) {      // log Q = -log1p(listed / unlisted); beyond exp(600) the 1 is lost anyway
            const double d = ((double)in.m - (double)out.m) * A.inv_ts;
            loss += rest * (log1p(-mass) + (d > 600.0 ? d + log(in.z / out.z) : in.z > 0.0 ? log1p(in.z / out.z * exp(d)) : 0.0));
        }
        const double inside = (mass + rest) / all.z;
        o.m = all.m;
        o.inside = (float)inside;
        o.m_out = out.m == -INFINITY ? 0.f : out.m;
        o.outside = with_rest ? (float)(inside * exp(((double)out.m - (double)all.m) * A.inv_ts) - (rest > 0.0 ? rest / out.z : 0.0))
                              : o.inside;
    }
    A.row[r] = o;
    A.loss[r] = any ? (float)loss : 0.f;
}

// sums of a workgroup's threads' (m, z), z in 32 bits; every thread receives the result
template <int TPB>
__device__ __forceinline__ MaxSum group_join(float m, float z, float c, float* s_m, double* s_z) {
    float top = group_max<64>(m);
    if constexpr (TPB > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) s_m[threadIdx.x >> 6] = top;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < TPB / 64; ++i) top = fmaxf(top, s_m[i]);
    }
    double zd = wave_sum(m == -INFINITY || m == top ? (double)z : (double)z * (double)exp_scaled(m - top, c));
    if constexpr (TPB > 64) {
        if ((threadIdx.x & 63) == 0) s_z[threadIdx.x >> 6] = zd;
        __syncthreads();
        zd = 0.0;
#pragma unroll
        for (int i = 0; i < TPB / 64; ++i) zd += s_z[i];
    }
    return {top, zd};
}

// One workgroup per (row, segment).
template <typename T, int TPB>
__global__ __launch_bounds__(TPB) void k_distill_fwd(DistillArgs A, float c) {
    constexpr int VEC = Elem<T>::VEC, GROUP = 4;
    __shared__ uint32_t s_bits[DISTILL_SEG / 32];
    __shared__ int s_twice;
    __shared__ float s_m[TPB / 64];
    __shared__ double s_z[TPB / 64];
    const int64_t r = blockIdx.x / A.segs;
    const int seg = (int)(blockIdx.x - r * A.segs);
    const int v0 = seg * DISTILL_SEG, n = min(A.V - v0, DISTILL_SEG);
    const T* row = (const T*)A.s + r * A.lds + v0;
    const bool mask = A.lse != nullptr;
    if (mask) segment_bitmap(A.idx + r * A.ldi, A.k, v0, v0 + n, s_bits, &s_twice);
    float m = -INFINITY, z = 0.f;
    for (int at = threadIdx.x * VEC; at < n; at += TPB * VEC * GROUP) {
        float v[GROUP][VEC];
        if (n >= VEC) {
            // all loads first; what is not a slot's own (see raw_slot) and what is listed does not count
            Slot<T> raw[GROUP];
            uint32_t dead[GROUP];
#pragma unroll
            for (int u = 0; u < GROUP; ++u) raw[u] = raw_slot(row, at + u * TPB * VEC, n);
            uint32_t any = 0;
#pragma unroll
            for (int u = 0; u < GROUP; ++u) {
                const int o = at + u * TPB * VEC, foreign = min(o - (int)slot_at<T>(o, n), VEC);
                dead[u] = (1u << foreign) - 1u;
                if (mask && o < n) dead[u] |= (s_bits[o >> 5] >> (o & 31)) << foreign;
                dead[u] &= (1u << VEC) - 1u;
                any |= dead[u];
            }
#pragma unroll
            for (int u = 0; u < GROUP; ++u)
#pragma unroll
                for (int i = 0; i < VEC; ++i) v[u][i] = (float)raw[u].v[i];
            if (any != 0) {
#pragma unroll
                for (int u = 0; u < GROUP; ++u)
#pragma unroll
                    for (int i = 0; i < VEC; ++i)
                        if ((dead[u] >> i) & 1u) v[u][i] = -INFINITY;
            }
        } else {
#pragma unroll
            for (int u = 0; u < GROUP; ++u) {
                load_slot(row, at + u * TPB * VEC, n, -INFINITY, v[u]);
                if (mask && u == 0) {
#pragma unroll
                    for (int i = 0; i < VEC; ++i)
                        if ((s_bits[0] >> (at + i)) & 1u) v[u][i] = -INFINITY;
                }
            }
        }
        float top = m;
#pragma unroll
        for (int u = 0; u < GROUP; ++u)
#pragma unroll
            for (int i = 0; i < VEC; ++i) top = fmaxf(top, v[u][i]);
        const float ref = top == -INFINITY ? 0.f : top;
        float sum = 0.f;
#pragma unroll
        for (int u = 0; u < GROUP; ++u)
#pragma unroll
            for (int i = 0; i < VEC; ++i) sum += exp_scaled(v[u][i] - ref, c);
        z = (m == -INFINITY ? z : z * exp_scaled(m - ref, c)) + sum;
        m = top;
    }
    const MaxSum out = group_join<TPB>(m, z, c, s_m, s_z);
    MaxSum in{-INFINITY, 0.0};
    if (mask) {          // the listed entries, each once: the set bits
        m = -INFINITY; z = 0.f;
        for (int w = threadIdx.x; w < (n + 31) / 32; w += TPB)
            for (uint32_t b = s_bits[w]; b != 0; b &= b - 1) {
                const float v = (float)row[w * 32 + __ffs(b) - 1], top = fmaxf(m, v), ref = top == -INFINITY ? 0.f : top;
                z = (m == -INFINITY ? z : z * exp_scaled(m - ref, c)) + exp_scaled(v - ref, c);
                m = top;
            }
        in = group_join<TPB>(m, z, c, s_m, s_z);
    }
    if (A.segs > 1) {
        if (threadIdx.x == 0) A.part[blockIdx.x] = make_float4(out.m, (float)out.z, in.m, (float)in.z);
    } else if (threadIdx.x < 64) {
        finish_row<T>(A, r, out, in);
    }
}

// rows cut into several segments: one wave per row joins them
template <typename T>
__global__ __launch_bounds__(64) void k_distill_join(DistillArgs A) {
    const int64_t r = blockIdx.x;
    MaxSum out{-INFINITY, 0.0}, in{-INFINITY, 0.0};
    for (int g = threadIdx.x; g < A.segs; g += 64) {
        const float4 q = A.part[r * A.segs + g];
        out = join(out, {q.x, (double)q.y}, A.inv_ts);
        in = join(in, {q.z, (double)q.w}, A.inv_ts);
    }
    finish_row<T>(A, r, wave_join(out, A.inv_ts), wave_join(in, A.inv_ts));
}

struct DistillBwdArgs {
    const void* s; int64_t lds; int V;
    const int64_t* idx; int64_t ldi; int k;
    const float* p; const DistillRow* row; const float* g;
    void* ds; float inv_t; int segs;
    template <typename T> DistillBwdArgs from(int64_t r) const {
        DistillBwdArgs a = *this;
        a.s = (const T*)s + r * lds; a.idx += r * ldi; a.p += r * k; a.row += r; a.g += r; a.ds = (T*)ds + r * V;
        return a;
    }
};

// One workgroup per (row, segment): the stream first, then the listed entries over what it wrote (same workgroup, behind a
// barrier).  Entries of one index add up; each of them writes the same value.
template <typename T, int TPB>
__global__ __launch_bounds__(TPB) void k_distill_bwd(DistillBwdArgs A, float c) {
    constexpr int VEC = Elem<T>::VEC, GROUP = 2;
    __shared__ uint32_t s_bits[DISTILL_SEG_BWD / 32];
    __shared__ int s_twice;
    const int64_t r = blockIdx.x / A.segs;
    const int seg = (int)(blockIdx.x - r * A.segs);
    const int v0 = seg * DISTILL_SEG_BWD, n = min(A.V - v0, DISTILL_SEG_BWD);
    const T* row = (const T*)A.s + r * A.lds + v0;
    T* out = (T*)A.ds + r * (int64_t)A.V + v0;
    const DistillRow R = A.row[r];
    const bool live = !(R.inside == 0.f && R.outside == 0.f);
    const float g = live ? A.g[r] * A.inv_t : 0.f;
    const float fo = g * R.outside, fi = g * R.inside;
    for (int at = threadIdx.x * VEC; at < n; at += TPB * VEC * GROUP) {
        if (n >= VEC) {
            // (a slot that was moved back writes some of its neighbour's results once more)
            Slot<T> raw[GROUP];
            if (live) {
#pragma unroll
                for (int u = 0; u < GROUP; ++u) raw[u] = raw_slot(row, at + u * TPB * VEC, n);
            }
#pragma unroll
            for (int u = 0; u < GROUP; ++u) {
                const int o = at + u * TPB * VEC;
                Slot<T> r;
#pragma unroll
                for (int i = 0; i < VEC; ++i) r.v[i] = (T)(live ? exp_scaled((float)raw[u].v[i] - R.m_out, c) * fo : 0.f);
                if (o < n) *reinterpret_cast<Slot<T>*>(out + slot_at<T>(o, n)) = r;
            }
        } else {
            float v[VEC];
            if (live) load_slot(row, at, n, -INFINITY, v);
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[i] = live ? exp_scaled(v[i] - R.m_out, c) * fo : 0.f;
            store_slot(out, at, n, v);
        }
    }
    if (!live) return;
    const int64_t* idx = A.idx + r * A.ldi;
    const bool twice = segment_bitmap(idx, A.k, v0, v0 + n, s_bits, &s_twice);
    for (int j = threadIdx.x; j < A.k; j += TPB) {
        const int64_t i = idx[j];
        if (i < v0 || i >= v0 + n) continue;
        float p = 0.f;
        if (!twice) p = A.p[r * A.k + j];
        else
            for (int e = 0; e < A.k; ++e)
                if (idx[e] == i) p += A.p[r * A.k + e];
        out[i - v0] = (T)(exp_scaled((float)row[i - v0] - R.m, c) * fi - g * p);
    }
}

static inline int distill_segs(int V, int seg = DISTILL_SEG) { return V / seg + (V % seg != 0); }

static float distill_factor(double temperature) { return (float)(1.4426950408889634074 / temperature); }

static int distill_check(const char* what, const void* s, int64_t lds, int dtype, const void* idx, int64_t ldi, int64_t rows,
                         int32_t V, int32_t k, double temperature) {
    DRM_REQUIRE(s && (idx || k == 0), DRM_EINVAL, "%s: null pointer", what);
    DRM_REQUIRE(elem_ok(dtype), DRM_ENOTSUP, "%s: element type %d (fp32, bf16 or fp16)", what, dtype);
    DRM_REQUIRE(rows >= 0 && V >= 1 && lds >= V, DRM_EINVAL, "%s: rows=%lld V=%d row stride %lld", what, (long long)rows, V, (long long)lds);
    DRM_REQUIRE(k >= 0 && ldi >= k, DRM_EINVAL, "%s: k=%d list stride %lld", what, k, (long long)ldi);
    DRM_REQUIRE(k <= DISTILL_MAX_K, DRM_ENOTSUP, "%s: k=%d listed entries (at most %d)", what, k, DISTILL_MAX_K);
    DRM_REQUIRE(temperature > 0.0 && temperature <= 1e6 && temperature >= 1e-6, DRM_EINVAL, "%s: temperature %g", what, temperature);
    DRM_REQUIRE(rows <= INT_MAX / distill_segs(V, DISTILL_SEG_BWD), DRM_ENOTSUP, "%s: %lld rows of %d entries", what, (long long)rows, V);
    return DRM_OK;
}

}  // namespace drm

using namespace drm;

extern "C" size_t drm_distill_topk_workspace_bytes(int64_t rows, int32_t V) {
    if (rows < 0 || V < 1 || distill_segs(V) == 1) return 0;
    return (size_t)rows * distill_segs(V) * sizeof(float4);
}

extern "C" int drm_distill_topk_forward(const void* logits, int64_t ld_logits, int32_t dtype, const float* top_values, int64_t ld_values,
                                        const int64_t* top_indices, int64_t ld_indices, const float* top_lse, int64_t rows, int32_t V,
                                        int32_t k, double temperature, float* loss, float* p_out, float* row_out, void* workspace,
                                        size_t workspace_bytes, drm_stream_t stream) {
    if (rows == 0) return DRM_OK;
    if (int rc = distill_check(__func__, logits, ld_logits, dtype, top_indices, ld_indices, rows, V, k, temperature)) return rc;
    DRM_REQUIRE(loss && row_out && ((top_values && p_out) || k == 0) && ld_values >= k, DRM_EINVAL, "null pointer or list stride %lld below k=%d",
                (long long)ld_values, k);
    DRM_REQUIRE(aligned16(row_out), DRM_EINVAL, "row_out must be 16-byte aligned");
    const size_t need = drm_distill_topk_workspace_bytes(rows, V);
    DRM_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && aligned16(workspace)), DRM_EINVAL,
                "workspace of %zu bytes, %zu needed (16-byte aligned)", workspace ? workspace_bytes : (size_t)0, need);
    hipStream_t s = (hipStream_t)stream;
    const float c = distill_factor(temperature);
    DistillArgs A{logits, ld_logits, V, top_values, ld_values, top_indices, ld_indices, k, top_lse, 1.0 / temperature,
                  (double)c * 0.69314718055994530942, distill_segs(V), (float4*)workspace, loss, p_out, (DistillRow*)row_out};
    const double n = (double)rows * V;
    ProfScope ps(PC_ELEMENTWISE, s, 6 * n, n * elem_bytes(dtype) + (double)rows * k * 12);
    return with_elem(dtype, [&](auto tag) -> int {
        using T = decltype(tag);
        // one wave a row: more rows under way (8192 x 4096 bf16 22 us, four waves a row 34); few longer rows want the four (256 x
        // 8192: 7.5 and 5.8 us)
        const int64_t most = launch_limit(V <= 4096 ? 64 : 256) / A.segs;
        for (int64_t r = 0; r < rows; r += most) {
            const DistillArgs P = A.from<T>(r);
            const int grid = (int)(std::min(rows - r, most) * A.segs);
            if (V <= 4096) k_distill_fwd<T, 64><<<grid, 64, 0, s>>>(P, c);
            else k_distill_fwd<T, 256><<<grid, 256, 0, s>>>(P, c);
            DRM_LAUNCH_CHECK();
        }
        if (A.segs > 1) {
            k_distill_join<T><<<(int)rows, 64, 0, s>>>(A);
            DRM_LAUNCH_CHECK();
        }
        return DRM_OK;
    });
}

extern "C" int drm_distill_topk_backward(const void* logits, int64_t ld_logits, int32_t dtype, const int64_t* top_indices,
                                         int64_t ld_indices, const float* p, const float* row, const float* g_rows,
                                         int64_t rows, int32_t V, int32_t k, double temperature, void* d_logits, drm_stream_t stream) {
    if (rows == 0) return DRM_OK;
    if (int rc = distill_check(__func__, logits, ld_logits, dtype, top_indices, ld_indices, rows, V, k, temperature)) return rc;
    DRM_REQUIRE(row && g_rows && d_logits && (p || k == 0), DRM_EINVAL, "null pointer");
    DRM_REQUIRE(aligned16(row), DRM_EINVAL, "row must be 16-byte aligned");
    hipStream_t s = (hipStream_t)stream;
    const float c = distill_factor(temperature);
    DistillBwdArgs A{logits, ld_logits, V, top_indices, ld_indices, k, p, (const DistillRow*)row, g_rows, d_logits,
                     (float)(1.0 / temperature), distill_segs(V, DISTILL_SEG_BWD)};
    const double n = (double)rows * V;
    ProfScope ps(PC_ELEMENTWISE, s, 5 * n, 2 * n * elem_bytes(dtype) + (double)rows * k * 12);
    return with_elem(dtype, [&](auto tag) -> int {
        using T = decltype(tag);
        // (32768 x 1024 bf16: one wave 30 us, four 46; 1024 x 4096: 6.5 and 5.3)
        const int64_t most = launch_limit(V <= 2048 ? 64 : 256) / A.segs;
        for (int64_t r = 0; r < rows; r += most) {
            const DistillBwdArgs P = A.from<T>(r);
            const int grid = (int)(std::min(rows - r, most) * A.segs);
            if (V <= 2048) k_distill_bwd<T, 64><<<grid, 64, 0, s>>>(P, c);
            else k_distill_bwd<T, 256><<<grid, 256, 0, s>>>(P, c);
            DRM_LAUNCH_CHECK();
        }
        return DRM_OK;
    });
}
