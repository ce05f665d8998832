// Microscaled 4-bit floating point: quantisation, its inverse, and the products that read 4-bit weights.
#include "colsum.hpp"
#include "mx4.hpp"

#include <algorithm>
#include <climits>
#include <type_traits>

namespace drm {

// ---- quantisation -------------------------------------------------------------------------------------------------------
// e = floor(log2(max |x|)) - 2, clamped to [-127, 127]; code = x / 2^e rounded to the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6 (ties
// to the even code), 6 beyond.  Four lanes share a block: eight elements, four code bytes each.  A stream: bound by the bytes
// (12288 x 4096 bf16 20 us, 6.5 TB/s; 16384 x 8192 fp32 115 us, 5.3 TB/s).
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

// A lane writes one 16-byte slot of the row (VEC codes): 12288 x 4096 bf16 20 us (6.4 TB/s); a block a lane, whose writes lie 64
// bytes apart, took 31 us.
template <typename T>
__global__ __launch_bounds__(256) void k_mx4_dequantize(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int64_t rows,
                                                        int K, int nb, T* __restrict__ y, int64_t ldy) {
    constexpr int VEC = Elem<T>::VEC, PER = 32 / VEC;
    using Codes = std::conditional_t<VEC == 8, uint32_t, uint16_t>;
    const int64_t slots = rows * nb * PER, step = (int64_t)gridDim.x * 256;
    for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < slots; q += step) {
        const int64_t blk = q / PER, r = blk / nb;
        // bf16 holds every value; below 2^128 so do fp32 and, inside its range, fp16
        const bf16x8 h = mx4_bf16x8((uint32_t)reinterpret_cast<const Codes*>(codes)[q], mx4_scale(scales[blk]));
        float v[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = (float)h[i];
        store_slot(y + r * ldy, (blk - r * nb) * 32 + (q % PER) * VEC, K, v);
    }
}

// Workgroup -> output tile.  Workgroups go round the eight XCDs, each with an L2 of its own: every XCD gets a run of consecutive
// tiles in an order that walks columns of eight row tiles, so that the tiles in flight on it share rows and columns.
__device__ __forceinline__ void mx4_tile_of(int id, int tiles_m, int tiles_n, int& tm, int& tn) {
    const int total = tiles_m * tiles_n, per = total / 8, extra = total % 8, xcd = id % 8;
    const int pos = xcd * per + min(xcd, extra) + id / 8;
    const int group = 8 * tiles_n, g = pos / group, first = g * 8, rows = min(8, tiles_m - first);
    tm = first + (pos - g * group) % rows;
    tn = (pos - g * group) / rows;
}

// what lies behind the last block of a row: sixteen zero bytes in memory
__device__ const uint4 mx4_zero_block = {0u, 0u, 0u, 0u};

// ---- y = x W^T + bias, few rows -----------------------------------------------------------------------------------------
// The weight is streamed once.  A workgroup takes 16 NT weight rows, its NW waves share the reduction in passes of four blocks (128
// elements).  In the matrix instruction lanes 0-15 are sixteen rows, so fragments read straight from memory would touch a cache
// line per lane, and the address path, at a line a clock, would take three times the time of the bytes.  Each wave therefore
// brings its pass to LDS of its own by direct loads (16 weight rows of 64 bytes, MT x 16 rows of x), two passes under way, and
// reads the fragments there.  A lane holds one block of a weight row and feeds it to four instructions, eight elements at a
// time; the four lane groups hold different blocks, a permutation of the reduction index that x follows.  x comes from L2 for every
// workgroup, which is why a wave takes NT weight tiles to one fragment of x.  The waves' sums meet in LDS in a fixed order.
// Bound by the weight's bytes: 16 x 12288 x 4096 bf16 9.4 us (2.9 TB/s; an empty launch takes 3 us of it), 16 x 8192 x 8192 10.5 us
// (3.4 TB/s).  fp32 rows have three parts, three times the instructions and the x traffic: 16 x 12288 x 4096 17 us
// (fp16, two parts: 11.5 us).  Times here and below: recorded graph of twenty calls in a row, per call.
template <typename T, int MT, int NT, int NW>
struct RowsStage {
    __attribute__((aligned(16))) uint8_t w[NW][NT * 1024], x[NW][MT * 16 * 128 * sizeof(T)];
    uint32_t sc[NW][NT * 64];
};

template <int N>
__device__ __forceinline__ void wait_loads() {        // no more than N vector memory operations under way, LDS reads done
    static_assert(N < 64);
    __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 0x0070);
    asm volatile("" ::: "memory");
}

// A barrier behind which every wave finds what the others brought to LDS: direct loads count as vector memory operations.
__device__ __forceinline__ void stage_barrier() {
    wait_loads<0>();
    __syncthreads();
}

template <typename T, int MT, int NT, int NW>
__device__ __forceinline__ void mx4_rows_store(f32x4* s_acc, const f32x4 (&acc)[NT][MT], const Mx4& W, const void* bias, int btype,
                                               T* __restrict__ y, int64_t ldy, int M, int n0) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int t = 0; t < MT; ++t) s_acc[((w * NT + i) * MT + t) * 64 + lane] = acc[i][t];
    __syncthreads();
    for (int o = threadIdx.x; o < NT * MT * 64; o += NW * 64) {
        const int i = o / (MT * 64), t = (o >> 6) % MT, l = o & 63;
        f32x4 v = s_acc[o];
#pragma unroll
        for (int k = 1; k < NW; ++k) v += s_acc[k * NT * MT * 64 + o];
        const int m = t * 16 + (l & 15), nn = n0 + i * 16 + 4 * (l >> 4);
        if (m < M)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (nn + e < W.rows) y[m * ldy + nn + e] = (T)(v[e] + (bias != nullptr ? load_elem(bias, btype, nn + e) : 0.f));
    }
}

template <typename T, int MT, int NT, int NW>
__global__ __launch_bounds__(NW * 64) void k_mx4_rows(const T* __restrict__ x, int64_t ldx, Mx4 W, const void* bias, int btype,
                                                      T* __restrict__ y, int64_t ldy, int M, int K) {
    constexpr int P = Parts<T>::N, EPC = 16 / sizeof(T), XCH = 128 / EPC, XI = MT * 16 * XCH / 64, LOADS = 2 * NT + XI;
    using Stage = RowsStage<T, MT, NT, NW>;
    __shared__ Stage s0, s1;
    static_assert(sizeof(Stage) >= NW * NT * MT * 64 * sizeof(f32x4), "the waves' sums fit one stage");
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, g = lane >> 4, c = lane & 15;
    const int n0 = blockIdx.x * 16 * NT;
    f32x4 acc[NT][MT];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[i][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int turns = ((W.nb + 3) / 4 + NW - 1) / NW;          // this wave's passes: w, w + NW, ...; behind the last block: zero blocks
    auto issue = [&](Stage& st, int i) {
        asm volatile("" ::: "memory");
        const int base = (w + i * NW) * 4;
        // a lane's own scale byte of each weight tile, widened to a dword by the load
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const uint8_t* src = W.scales + (int64_t)min(n0 + t * 16 + c, W.rows - 1) * W.nb + min(base + g, W.nb - 1);
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) uint32_t*)src,
                                             (__attribute__((address_space(3))) uint32_t*)(st.sc[w] + t * 64), 1, 0, 0);
        }
        // slot p of weight row r holds block p ^ (r / 4): sixteen rows of one block lie on different banks
        const int wr = lane >> 2, kb = base + ((lane & 3) ^ ((wr >> 2) & 3));
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const uint8_t* src = W.codes + ((int64_t)min(n0 + t * 16 + wr, W.rows - 1) * W.nb + kb) * 16;
            src = kb < W.nb ? src : reinterpret_cast<const uint8_t*>(&mx4_zero_block);
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) uint32_t*)src,
                                             (__attribute__((address_space(3))) uint32_t*)(st.w[w] + t * 1024), 16, 0, 0);
        }
#pragma unroll
        for (int j = 0; j < XI; ++j) {
            const int slot = j * 64 + lane, r = slot / XCH, p = slot % XCH, k = base * 32 + ((p & 16) | ((p ^ r) & 15)) * EPC;
            const uint8_t* src = reinterpret_cast<const uint8_t*>(x + (int64_t)min(r, M - 1) * ldx + k);
            src = k < K ? src : reinterpret_cast<const uint8_t*>(&mx4_zero_block);
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) uint32_t*)src,
                                             (__attribute__((address_space(3))) uint32_t*)(st.x[w] + j * 1024), 16, 0, 0);
        }
        asm volatile("" ::: "memory");
    };
    auto compute = [&](const Stage& st) {
        u32x4 q[NT];
        float sc[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) sc[i] = mx4_scale(st.sc[w][i * 64 + lane]);
#pragma unroll
        for (int i = 0; i < NT; ++i) q[i] = *reinterpret_cast<const u32x4*>(st.w[w] + i * 1024 + c * 64 + ((g ^ ((c >> 2) & 3)) * 16));
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            bf16x8 a[NT];
#pragma unroll
            for (int i = 0; i < NT; ++i) a[i] = mx4_bf16x8(q[i][s], sc[i]);
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                Eight<T> e;
#pragma unroll
                for (int h = 0; h < 8 / EPC; ++h) {
                    const int ch = (g * 32 + s * 8) / EPC + h;
                    reinterpret_cast<u32x4*>(&e)[h] = *reinterpret_cast<const u32x4*>(st.x[w] + ((t * 16 + c) * XCH + ((ch & 16) | ((ch ^ c) & 15))) * 16);
                }
                bf16x8 b[P];
                split_eight<T>(e, b);
#pragma unroll
                for (int p = P - 1; p >= 0; --p)
#pragma unroll
                    for (int i = 0; i < NT; ++i) acc[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[p], acc[i][t], 0, 0, 0);
            }
        }
    };
    issue(s0, 0);
    if (turns == 1) {
        wait_loads<0>();
        compute(s0);
    } else {
        issue(s1, 1);
        for (int i = 0; i + 2 < turns; i += 2) {
            wait_loads<LOADS>();              // the other stage's loads may still be under way
            compute(s0);
            wait_loads<63>();
            issue(s0, i + 2);
            wait_loads<LOADS>();
            compute(s1);
            wait_loads<63>();
            issue(s1, i + 3);
        }
        wait_loads<LOADS>();
        compute(s0);
        wait_loads<0>();
        compute(s1);
    }
    __syncthreads();
    mx4_rows_store<T, MT, NT, NW>(reinterpret_cast<f32x4*>(&s0), acc, W, bias, btype, y, ldy, M, n0);
}

// The same product for rows of x that direct loads cannot take (not aligned to 16 bytes, or not whole chunks): fragments from memory,
// a cache line a lane (16 x 4096 x 4096 bf16 16.5 us; aligned rows above 5.0 us).
template <typename T, int MT, int NW>
__global__ __launch_bounds__(NW * 64) void k_mx4_rows_any(const T* __restrict__ x, int64_t ldx, Mx4 W, const void* bias, int btype,
                                                          T* __restrict__ y, int64_t ldy, int M, int K) {
    constexpr int P = Parts<T>::N;
    __shared__ f32x4 s_acc[NW * MT * 64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, g = lane >> 4, c = lane & 15;
    const int n0 = blockIdx.x * 16;
    const int64_t row = (int64_t)min(n0 + c, W.rows - 1) * W.nb;
    f32x4 acc[1][MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[0][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int base = w * 4; base < W.nb; base += NW * 4) {
        const int kb = base + g;
        const bool live = kb < W.nb;                     // a block behind the last one: zero codes at scale 1
        const u32x4 q = reinterpret_cast<const u32x4*>(W.codes)[row + min(kb, W.nb - 1)];
        const float sc = mx4_scale(live ? W.scales[row + min(kb, W.nb - 1)] : 127u);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const bf16x8 a = mx4_bf16x8(live ? q[s] : 0u, sc);
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                bf16x8 b[P];
                load_parts(x + (int64_t)min(t * 16 + c, M - 1) * ldx, (int64_t)kb * 32 + s * 8, K, b);
#pragma unroll
                for (int p = P - 1; p >= 0; --p) acc[0][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b[p], acc[0][t], 0, 0, 0);
            }
        }
    }
    mx4_rows_store<T, MT, 1, NW>(s_acc, acc, W, bias, btype, y, ldy, M, n0);
}

// A row's NB blocks of a step in LDS: block b in slot b ^ (the row's number), so that eight rows of one block fall on all banks
template <int NB>
__device__ __forceinline__ int mx4_code_slot(int r, int b) { return NB == 4 ? b ^ ((r >> 1) & 3) : b ^ ((r >> 2) & 1); }

// Outputs of a wave (WM rows x WN columns in 32x32 accumulators whose lanes are rows): 32 rows at a time turn through LDS, so that
// they leave in 16-byte pieces of a row.  `strip`: 32 x (WN + 4) floats of this wave's own.
template <typename T, int WM, int WN>
__device__ __forceinline__ void mx4_store_tile(float* strip, const f32x16 (&acc)[WN / 32][WM / 32], T* __restrict__ y, int64_t ldy, int m0,
                                               int n0, int M, int N, const void* bias, int btype) {
    constexpr int LD = WN + 4, VEC = Elem<T>::VEC, LPR = WN / VEC;             // lanes per row
    const int lane = threadIdx.x & 63, nl = (lane % LPR) * VEC, n = n0 + nl;
    float bv[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) bv[i] = bias != nullptr && n + i < N ? load_elem(bias, btype, n + i) : 0.f;
#pragma unroll
    for (int j = 0; j < WM / 32; ++j) {
#pragma unroll
        for (int i = 0; i < WN / 32; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                *reinterpret_cast<f32x4*>(&strip[(lane & 31) * LD + i * 32 + 8 * q + 4 * (lane >> 5)]) =
                    f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
        __builtin_amdgcn_wave_barrier();        // one wave's LDS accesses stay in order
#pragma unroll
        for (int r = 0; r < 32; r += 64 / LPR) {
            const int row = r + lane / LPR, m = m0 + j * 32 + row;
            float v[VEC];
#pragma unroll
            for (int i = 0; i < VEC; i += 4) {
                const f32x4 f = *reinterpret_cast<const f32x4*>(&strip[row * LD + nl + i]);
                v[i] = f[0] + bv[i]; v[i + 1] = f[1] + bv[i + 1]; v[i + 2] = f[2] + bv[i + 2]; v[i + 3] = f[3] + bv[i + 3];
            }
            if (m < M && n < N) store_slot(y + m * ldy, n, N, v);
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// ---- y = x W^T + bias and dx = dy W, many rows --------------------------------------------------------------------------
// 128 x 128 outputs per workgroup, eight waves of 64 x 32 (32x32x16 bf16 matrix instructions), BK of the reduction per step, two or
// three LDS stages.  Eight waves although four larger ones would read less from LDS: a single wave of a SIMD issues a vector
// instruction every eight cycles only, two of them every four.  The float operand lies in LDS in its bf16 parts: rows of BK,
// 16-byte chunks in an order that spreads a fragment's rows over the banks; bf16 rows whose chunks are aligned go there by direct
// loads, others through registers.
//   y : the codes lie in LDS as they are and every wave widens the fragments it needs (a quarter of the LDS traffic of bf16
//       rows, for one conversion per two elements, at the rate of ordinary vector instructions, under the matrix instructions).
//   dx: the reduction runs over W's rows, so that a fragment needs one column of eight rows: the block of a row is widened
//       once, four rows side by side exchange their dwords (a transposition among four lanes), and the columns go to LDS.
// bf16, y / dx: 1024 x 4096 x 4096 42 / 47 us (830 TFLOP/s; a library product of the same size with a bf16 weight 39 / 45 us),
// 2048 x 8192 x 4096 145 / 161 us (950).  fp16 rows have two parts (81 / 88 us), fp32 rows three (116 / 117 us).  Bound by the
// issue of vector and LDS instructions between the matrix instructions, which are busy a third of the time.
constexpr int TILE_WAVES = 8, TILE_THREADS = TILE_WAVES * 64;
template <typename T, int BK, bool GRAD>
struct TileStage {
    static constexpr int P = Parts<T>::N, NB = BK / 32;
    __attribute__((aligned(16))) uint8_t x[P][128 * BK * 2];
    __attribute__((aligned(16))) uint8_t w[GRAD ? 128 * BK * 2 : 128 * NB * 16];
    uint32_t sw[GRAD ? 4 : TILE_THREADS];  // 128 rows (brought by every pair of waves)
};

// Position of chunk c in row r of a tile of bf16 rows of CH chunks: the sixteen rows that one clock of a fragment read takes
// (64 banks, 256 bytes) lie on different banks.  An involution in c.
template <int CH>
__device__ __forceinline__ int mx4_chunk(int r, int c) { return CH == 16 ? c ^ (r & 15) : c ^ ((r >> 1) & 7); }
// dx: columns of W; the lanes of one instruction write columns whose numbers differ by eight, so r / 8 takes part as well
template <int CH>
__device__ __forceinline__ int mx4_chunk_t(int r, int c) { return CH == 16 ? c ^ ((r ^ (r >> 3)) & 15) : c ^ (((r >> 1) ^ (r >> 3)) & 7); }

struct __attribute__((packed, aligned(1))) Bytes4 { uint32_t v; };
struct __attribute__((packed, aligned(1))) Bytes2 { uint16_t v; };

template <int CTRL>
__device__ __forceinline__ uint32_t quad(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false); }

// One block (16 bytes) of each of four rows that sit in the four lanes of a quad -> lane q: codes 8 q .. 8 q + 7 of the four rows
__device__ __forceinline__ u32x4 quad_transpose(u32x4 d, int q) {
    const bool odd = q & 1, high = q & 2;
    uint32_t t0 = quad<0xB1>(odd ? d[0] : d[1]), t1 = quad<0xB1>(odd ? d[2] : d[3]);
    if (odd) { d[0] = t0; d[2] = t1; } else { d[1] = t0; d[3] = t1; }
    t0 = quad<0x4E>(high ? d[0] : d[2]);
    t1 = quad<0x4E>(high ? d[1] : d[3]);
    if (high) { d[0] = t0; d[1] = t1; } else { d[2] = t0; d[3] = t1; }
    return d;
}

template <typename T, int BK, bool DIRECT, bool GRAD, bool RING>
__global__ __launch_bounds__(TILE_THREADS) void k_mx4_tile(const T* __restrict__ x, int64_t ldx, Mx4 W, const void* bias, int btype,
                                                  T* __restrict__ y, int64_t ldy, int M, int N, int K, int tiles_m, int tiles_n,
                                                  float* __restrict__ part, int span) {
    // y: reduction over W's columns (K of them), N = W's rows; dx: reduction over W's rows (K of them), N = W's columns
    // With `part` the workgroups of blockIdx.y take `span` of the reduction each and leave (gridDim.y, M, N) fp32 sums there.
    static_assert(!DIRECT || Parts<T>::N == 1, "direct loads bring bf16");
    static_assert(!RING || (DIRECT && !GRAD), "a ring of stages has no loads through registers");
    using Stage = TileStage<T, BK, GRAD>;
    constexpr int P = Stage::P, NB = Stage::NB, CH = BK / 8, XU = 128 * CH / TILE_THREADS, WU = GRAD ? BK * 4 / TILE_THREADS + (BK * 4 < TILE_THREADS) : 1;
    constexpr int WN = 32, OUT_LD = WN + 4;
    static_assert(sizeof(Stage) >= TILE_WAVES * 32 * OUT_LD * sizeof(float), "the output strips fit one stage");
    __shared__ Stage s0, s1;
    __shared__ std::conditional_t<RING, Stage, char> s2;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, l32 = lane & 31;
    int tm, tn;
    mx4_tile_of(blockIdx.x, tiles_m, tiles_n, tm, tn);
    const int m0 = tm * 128, n0 = tn * 128, wm = (wave & 1) * 64, wn = (wave >> 1) * WN;
    const int begin = blockIdx.y * span;                          // a multiple of BK
    K = min(K, begin + span);
    f32x16 acc[1][2];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[0][j][e] = 0.f;

    struct Held {                     // what a step brings through registers
        Eight<T> x[DIRECT ? 1 : XU];
        u32x4 w[WU];
        uint32_t sw[WU];
    };
    auto load_scales = [&](int k0, Held& h) {       // W.nb >= NB: the row's bytes of this step, or its last ones, shifted by put
        const uint8_t* p = W.scales + (int64_t)min(n0 + (int)(threadIdx.x & 127), N - 1) * W.nb + min(k0 >> 5, W.nb - NB);
        if constexpr (NB == 4) h.sw[0] = reinterpret_cast<const Bytes4*>(p)->v;
        else h.sw[0] = reinterpret_cast<const Bytes2*>(p)->v;
    };
    const int whole = DIRECT ? K : K & ~7;        // elements of a row in whole chunks (direct loads: all of them)
    auto load = [&](Stage& st, int k0, Held& h, bool tail) {
        if constexpr (GRAD) {
#pragma unroll
            for (int j = 0; j < WU; ++j) {
                const int u = (threadIdx.x + TILE_THREADS * j) & (BK * 4 - 1), n = k0 + (u >> 4) * 4 + (u & 3), kb = (n0 >> 5) + ((u >> 2) & 3);
                const int64_t at = (int64_t)min(n, W.rows - 1) * W.nb + min(kb, W.nb - 1);
                h.sw[j] = W.scales[at];
                h.w[j] = reinterpret_cast<const u32x4*>(W.codes)[at];
            }
        }
        if constexpr (DIRECT) {
            constexpr int RPI = 64 / CH;                          // rows per wave and instruction
            const int row = lane / CH;
            const uint8_t* base = reinterpret_cast<const uint8_t*>(x + (int64_t)m0 * ldx + k0);
#pragma unroll
            for (int j = 0; j < 128 / RPI / TILE_WAVES; ++j) {
                const int r = (j * TILE_WAVES + wave) * RPI + row;
                const int cc = mx4_chunk<CH>(r, lane % CH);
                const uint8_t* src = base + (uint32_t)(min(r, M - 1 - m0) * (int)ldx * 2 + cc * 16);
                src = k0 + cc * 8 < K ? src : reinterpret_cast<const uint8_t*>(&mx4_zero_block);
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) uint32_t*)src,
                                                 (__attribute__((address_space(3))) uint32_t*)(st.x[0] + (j * TILE_WAVES + wave) * 1024), 16, 0, 0);
            }
        } else {
            // whole chunks of eight; what is left of a row behind them follows in a step of its own
            if (!tail) {
#pragma unroll
                for (int j = 0; j < XU; ++j) {
                    const int u = threadIdx.x + TILE_THREADS * j, r = u / CH, c = u % CH;
                    h.x[j] = reinterpret_cast<const Packed8<T>*>(x + (int64_t)min(m0 + r, M - 1) * ldx + max(min(k0 + c * 8, whole - 8), 0))->e;
                }
            } else {
#pragma unroll
                for (int j = 0; j < XU; ++j) {
                    const int u = threadIdx.x + TILE_THREADS * j, r = u / CH, c = u % CH;
                    h.x[j] = load_eight(x + (int64_t)min(m0 + r, M - 1) * ldx, k0 + c * 8 < whole ? (int64_t)K : (int64_t)k0 + c * 8, K);
                }
            }
        }
        if constexpr (!GRAD) {
            const uint8_t* base = W.codes + ((int64_t)n0 * W.nb + (k0 >> 5)) * 16;
#pragma unroll
            for (int j = 0; j < (NB * 2 + TILE_WAVES - 1) / TILE_WAVES; ++j) {
                if (NB * 2 < TILE_WAVES && wave >= NB * 2) break;      // 64 per step: four waves bring the codes
                const int r = (j * TILE_WAVES + wave) * (64 / NB) + lane / NB, b = mx4_code_slot<NB>(r, lane % NB);
                const uint8_t* src = base + (uint32_t)((min(r, N - 1 - n0) * W.nb + b) * 16);
                src = (k0 >> 5) + b < W.nb ? src : reinterpret_cast<const uint8_t*>(&mx4_zero_block);
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) uint32_t*)src,
                                                 (__attribute__((address_space(3))) uint32_t*)(st.w + (j * TILE_WAVES + wave) * 1024), 16, 0, 0);
            }
        }
    };
    auto put = [&](Stage& st, int k0, const Held& h, bool tail) {
        if constexpr (!DIRECT) {
#pragma unroll
            for (int j = 0; j < XU; ++j) {
                const int u = threadIdx.x + TILE_THREADS * j, r = u / CH, c = u % CH;
                bf16x8 p[P];
                split_eight<T>(tail || k0 + c * 8 < whole ? h.x[j] : Eight<T>{}, p);
#pragma unroll
                for (int q = 0; q < P; ++q) *reinterpret_cast<bf16x8*>(st.x[q] + r * BK * 2 + mx4_chunk<CH>(r, c) * 16) = p[q];
            }
        }
        if constexpr (!GRAD) {
            const int kb0 = k0 >> 5;
            st.sw[threadIdx.x & 127] = h.sw[0] >> (min(kb0 - min(kb0, max(W.nb - NB, 0)), NB - 1) * 8);
        } else {
#pragma unroll
            for (int j = 0; j < WU; ++j) {
                const int u = threadIdx.x + TILE_THREADS * j, q = u & 3;
                if (BK * 4 < TILE_THREADS && u >= BK * 4) break;       // 64 per step: four waves put W away
                const bool live = k0 + (u >> 4) * 4 + q < W.rows && (n0 >> 5) + ((u >> 2) & 3) < W.nb;
                const u32x4 d = quad_transpose(live ? h.w[j] : u32x4{0u, 0u, 0u, 0u}, q);
                const uint32_t own = live ? h.sw[j] : 127u;
                const float sc[4] = {mx4_scale(quad<0x00>(own)), mx4_scale(quad<0x55>(own)), mx4_scale(quad<0xAA>(own)), mx4_scale(quad<0xFF>(own))};
                u32x4 r[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) r[i] = __builtin_bit_cast(u32x4, mx4_bf16x8(d[i], sc[i]));
                const int col = ((u >> 2) & 3) * 32 + q * 8, at = (u >> 4) * 4;     // eight columns, four rows of W
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint2 lo = make_uint2(__builtin_amdgcn_perm(r[1][i], r[0][i], 0x05040100u), __builtin_amdgcn_perm(r[3][i], r[2][i], 0x05040100u));
                    const uint2 hi = make_uint2(__builtin_amdgcn_perm(r[1][i], r[0][i], 0x07060302u), __builtin_amdgcn_perm(r[3][i], r[2][i], 0x07060302u));
                    const int c0 = col + 2 * i, c1 = c0 + 1;
                    *reinterpret_cast<uint2*>(st.w + c0 * BK * 2 + mx4_chunk_t<CH>(c0, at >> 3) * 16 + (at & 4) * 2) = lo;
                    *reinterpret_cast<uint2*>(st.w + c1 * BK * 2 + mx4_chunk_t<CH>(c1, at >> 3) * 16 + (at & 4) * 2) = hi;
                }
            }
        }
    };
    // A turn (16 of the reduction) fetches the next turn's fragments beside its own matrix instructions: x from LDS, the widened
    // codes of a block that was read a turn earlier.  (y: a lane half holds 16 codes in a row, eight per turn; dx: in order.)
    struct Turn { bf16x8 a, v[P][2]; };
    uint32_t sw = 0u;
    uint2 q[2];
    Turn f[2];
    const int wr = wn + l32;
    auto codes = [&](const Stage& st, int b) {
        if constexpr (!GRAD) {
            if (b == 0) sw = st.sw[wr];
            q[b & 1] = *reinterpret_cast<const uint2*>(st.w + wr * NB * 16 + mx4_code_slot<NB>(wr, b) * 16 + half * 8);
        }
    };
    auto fetch = [&](const Stage& st, int t) {
        const int b = t >> 1, c = GRAD ? t * 2 + half : b * 4 + half * 2 + (t & 1);
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int r = wm + j * 32 + l32;
                f[t & 1].v[p][j] = *reinterpret_cast<const bf16x8*>(st.x[p] + r * BK * 2 + mx4_chunk<CH>(r, c) * 16);
            }
        if constexpr (GRAD) f[t & 1].a = *reinterpret_cast<const bf16x8*>(st.w + wr * BK * 2 + mx4_chunk_t<CH>(wr, c) * 16);
        else f[t & 1].a = mx4_bf16x8((t & 1) == 0 ? q[b & 1].x : q[b & 1].y, mx4_scale((sw >> (8 * b)) & 255u));
    };
    auto multiply = [&](int t) {
#pragma unroll
        for (int p = P - 1; p >= 0; --p)
#pragma unroll
            for (int j = 0; j < 2; ++j)
                acc[0][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[t & 1].a, f[t & 1].v[p][j], acc[0][j], 0, 0, 0);
        // one matrix instruction, then the LDS reads and conversions of the next turn that fit beside it
#pragma unroll
        for (int k = 0; k < 2 * P; ++k) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, 3, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    auto compute = [&](const Stage& st) {
        codes(st, 0);
        fetch(st, 0);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int t = 0; t < 2 * NB; ++t) {
            if ((t & 1) == 0 && t / 2 + 1 < NB) codes(st, t / 2 + 1);
            if (t + 1 < 2 * NB) fetch(st, t + 1);
            multiply(t);
        }
    };
    Held h;
    if constexpr (!GRAD && !RING) {
        if (W.nb >= NB) {
            load_scales(begin, h);
        } else {                          // a row shorter than a step (then there is no second one)
            h.sw[0] = 0u;
            for (int i = 0; i < W.nb; ++i)
                h.sw[0] |= (uint32_t)W.scales[(int64_t)min(n0 + (int)(threadIdx.x & 127), N - 1) * W.nb + i] << (8 * i);
        }
    }
    const int steps = (max(whole - begin, 0) + BK - 1) / BK;
    if constexpr (RING) {
        // Three stages, filled by direct loads only (rows of whole steps of blocks: every row's four scale bytes of a step are an
        // aligned dword).  The waves meet before the last turn of a step, when all they need of its stage has been read: behind that
        // barrier the stage takes the loads of the step three ahead, the next one -- which every wave has waited for, leaving no more
        // than one later stage's loads under way (fences keep the loads of a stage together) -- gives its first fragments while
        // the last turn runs.
        constexpr int AHEAD = 128 * CH / TILE_THREADS + NB * 2 / TILE_WAVES + 1;
        static_assert(NB * 2 % TILE_WAVES == 0, "every wave brings as much");
        auto issue = [&](Stage& st, int k0) {
            asm volatile("" ::: "memory");
            const int kb0 = min(k0 >> 5, W.nb - NB);          // behind the last step: anything inside the row
            const uint8_t* src = W.scales + (int64_t)min(n0 + (int)(threadIdx.x & 127), N - 1) * W.nb + kb0;
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) uint32_t*)src,
                                             (__attribute__((address_space(3))) uint32_t*)(st.sw + wave * 64), 4, 0, 0);
            load(st, k0, h, false);
            asm volatile("" ::: "memory");
        };
        auto meet = [&](auto loads) {
            constexpr int L = decltype(loads)::value;
            __builtin_amdgcn_s_waitcnt((L & 15) | (L >> 4) << 14 | 0x0070);      // vmcnt(L), lgkmcnt(0)
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
        };
        auto step = [&](Stage& st, const Stage& next, int k0) {
#pragma unroll
            for (int t = 0; t + 1 < 2 * NB; ++t) {
                if ((t & 1) == 0 && t / 2 + 1 < NB) codes(st, t / 2 + 1);
                fetch(st, t + 1);
                multiply(t);
            }
            meet(std::integral_constant<int, AHEAD>{});
            issue(st, k0 + 3 * BK);
            codes(next, 0);
            fetch(next, 0);
            multiply(2 * NB - 1);
        };
        issue(s0, begin);
        issue(s1, begin + BK);
        issue(s2, begin + 2 * BK);
        meet(std::integral_constant<int, 2 * AHEAD>{});
        codes(s0, 0);
        fetch(s0, 0);
        int k0 = begin;
        for (int p = 0; p < steps / 3; ++p, k0 += 3 * BK) {
            step(s0, s1, k0);
            step(s1, s2, k0 + BK);
            step(s2, s0, k0 + 2 * BK);
        }
        if (steps % 3 > 0) step(s0, s1, k0);
        if (steps % 3 > 1) step(s1, s2, k0 + BK);
    } else if (steps > 0) {
        load(s0, begin, h, false);
        put(s0, begin, h, false);
        stage_barrier();
        for (int p = 0; p < steps / 2; ++p) {
            const int k1 = begin + (2 * p + 1) * BK, k2 = k1 + BK;
            if constexpr (!GRAD) load_scales(k1, h);      // first: nothing behind it has to wait for the rest
            load(s1, k1, h, false);
            compute(s0);
            put(s1, k1, h, false);
            stage_barrier();
            if constexpr (!GRAD) load_scales(k2, h);
            load(s0, k2, h, false);                       // behind the last step: not used
            compute(s1);
            put(s0, k2, h, false);
            stage_barrier();
        }
        if (steps & 1) compute(s0);
    }
    if (!DIRECT && whole < K) {
        const int k0 = max(whole / BK * BK, begin);
        if constexpr (!GRAD) { if (k0 > begin) load_scales(k0, h); }
        load(s1, k0, h, true);
        put(s1, k0, h, true);
        stage_barrier();
        compute(s1);
    }
    stage_barrier();
    float* strip = reinterpret_cast<float*>(&s0) + wave * 32 * OUT_LD;
    if (part != nullptr) mx4_store_tile<float, 64, WN>(strip, acc, part + (int64_t)blockIdx.y * M * N, N, m0 + wm, n0 + wn, M, N, nullptr, 0);
    else mx4_store_tile<T, 64, WN>(strip, acc, y, ldy, m0 + wm, n0 + wn, M, N, bias, btype);
}

// ---- both operands in 4 bits ----------------------------------------------------------------------------------------------
// Tiles of BM x BN outputs, 256 deep per step (eight blocks, 128 bytes a row), waves of WM x WN in 32x32x64 scaled
// matrix instructions.  The codes go from memory to LDS as they are (16-byte direct loads, no registers in between), two buffers:
// the loads of the next step run under the matrix instructions of this one.  A direct load fills LDS in lane order, so the lanes
// choose their source instead: slot p of row r holds block p ^ (r / 2 & 7): a fragment read takes 16 rows a clock, which then fall on all 64 banks.
// An instruction's lane half h takes block 4 h + s of the step's eight in its s-th turn -- a permutation of the reduction index that
// both operands share -- so that one dword holds a lane's four scales and the turn selects the byte.
// Blocks behind the last one come from the zero block, rows behind the last one repeat it and are not stored.
// 8192^3: 277 to 300 us in a row by the board and what ran before it (3.7 to 4.0 PFLOP/s; single calls under the profiler 282 to 340,
// 320 at the mean); 4096^3: 42 to 45 us, 3.2; 1024 x 4096 x 4096: 18 us, 1.9 (tiles of 128).  The instructions alone,
// from registers, reach 8.4 PFLOP/s with zeros but 5.7 to 6.5 with random codes, for which the clock falls (2.4 to below 2.0 GHz):
// that, not the nominal rate, is the ceiling.  Matrix instructions are busy 45 to 48% of the time; without the loads from memory the
// same loop takes 255 us, with a quarter of the LDS reads besides 214 us.
struct __attribute__((packed, aligned(1))) Bytes8 { uint32_t lo, hi; };

template <int BM, int BN>
struct ProductStage {
    __attribute__((aligned(16))) uint8_t x[BM * 128];
    __attribute__((aligned(16))) uint8_t w[BN * 128];
    uint32_t sx[BM * 2], sw[BN * 2];
    uint32_t room[512];                  // (the output strips of the smaller tiles are a little longer than their codes)
};

template <int ROWS, int WAVES>
__device__ __forceinline__ void mx4_stage_codes(const Mx4& A, int r0, int kb0, uint8_t* lds) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int lr = wave * 8 + (lane >> 3);
    asm volatile("" : "+v"(lr));            // offsets are formed at each step: kept, they would take the accumulators' registers
    const int c = (lane & 7) ^ (((wave * 8 + (lane >> 3)) >> 1) & 7), last = A.rows - 1 - r0;
    const uint8_t* base = A.codes + ((int64_t)r0 * A.nb + kb0) * 16;      // offsets inside a tile stay below 2^31 (checked at the call)
#pragma unroll
    for (int j = 0; j < ROWS / (8 * WAVES); ++j) {
        const uint8_t* src = base + (uint32_t)((min(lr + j * 8 * WAVES, last) * A.nb + c) * 16);
        src = kb0 + c < A.nb ? src : reinterpret_cast<const uint8_t*>(&mx4_zero_block);
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) uint32_t*)src,
                                         (__attribute__((address_space(3))) uint32_t*)(lds + (j * WAVES + wave) * 1024), 16, 0, 0);
    }
}
// the scale bytes of a row's blocks [kb0, kb0 + 8), 0 behind the last one; nb >= 8 (no branch: the row's last eight, shifted when
// they are put away, so that nothing waits for the load before)
__device__ __forceinline__ Bytes8 mx4_row_scales(const Mx4& A, int row, int kb0) {
    return *reinterpret_cast<const Bytes8*>(A.scales + (int64_t)min(row, A.rows - 1) * A.nb + min(kb0, A.nb - 8));
}
__device__ __forceinline__ uint2 mx4_shift_scales(Bytes8 b, int nb, int kb0) {
    const int shift = min(kb0 - min(kb0, nb - 8), 7) * 8;
    const uint64_t v = ((uint64_t)b.hi << 32 | b.lo) >> shift;
    return make_uint2((uint32_t)v, (uint32_t)(v >> 32));
}
// the same for a row of fewer than eight blocks
__device__ __forceinline__ uint2 mx4_short_row_scales(const Mx4& A, int row) {
    const uint8_t* p = A.scales + (int64_t)min(row, A.rows - 1) * A.nb;
    uint64_t v = 0;
    for (int i = 0; i < A.nb; ++i) v |= (uint64_t)p[i] << (8 * i);
    return make_uint2((uint32_t)v, (uint32_t)(v >> 32));
}

// fragments of turn S of a step, and the matrix instructions of a turn
template <int S, int TM, int TN>
__device__ __forceinline__ void mx4_turn_load(const uint8_t* x, const uint8_t* w, u32x4 (&b)[TM], u32x4 (&a)[TN]) {
    const int lane = threadIdx.x & 63;
    const int at = (lane & 31) * 128 + ((((lane >> 5) * 4 + S) ^ ((lane >> 1) & 7)) * 16);
#pragma unroll
    for (int i = 0; i < TN; ++i) a[i] = *reinterpret_cast<const u32x4*>(w + i * 32 * 128 + at);
#pragma unroll
    for (int j = 0; j < TM; ++j) b[j] = *reinterpret_cast<const u32x4*>(x + j * 32 * 128 + at);
}
__device__ __forceinline__ i32x8 mx4_operand(const u32x4& q) { return i32x8{(int)q[0], (int)q[1], (int)q[2], (int)q[3], 0, 0, 0, 0}; }
template <int S, int TM, int TN>
__device__ __forceinline__ void mx4_turn(const u32x4 (&b)[TM], const u32x4 (&a)[TN], const int (&sx)[TM], const int (&sw)[TN], f32x16 (&acc)[TN][TM]) {
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(mx4_operand(a[i]), mx4_operand(b[j]), acc[i][j], 4, 4, S, sw[i], S, sx[j]);
}

template <typename T, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__((BM / WM) * (BN / WN) * 64) void k_mx4_product(Mx4 X, Mx4 W, const void* bias, int btype, T* __restrict__ y, int64_t ldy, int tiles_m,
                                                     int tiles_n, float* __restrict__ part, int span) {
    // with `part` the workgroups of blockIdx.y take `span` steps of the reduction each and leave (gridDim.y, M, N) fp32 sums there
    constexpr int WAVES = (BM / WM) * (BN / WN), THREADS = WAVES * 64;
    constexpr int TM = WM / 32, TN = WN / 32;
    using Stage = ProductStage<BM, BN>;
    constexpr int OUT_LD = WN + 4;                                // floats per row of the output strip
    static_assert(sizeof(Stage) >= WAVES * 32 * OUT_LD * sizeof(float), "the output strips fit one stage");
    __shared__ Stage s0, s1;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int tm, tn;
    mx4_tile_of(blockIdx.x, tiles_m, tiles_n, tm, tn);
    const int m0 = tm * BM, n0 = tn * BN, wm = (wave / (BN / WN)) * WM, wn = (wave % (BN / WN)) * WN;
    f32x16 acc[TN][TM];
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    // scales: a thread brings those of one row of each tile, or of one of them where the threads suffice (smaller tiles: more than once)
    constexpr bool HALVES = THREADS >= BM + BN;
    const bool second = HALVES && threadIdx.x >= THREADS / 2;
    const int rx = threadIdx.x & (BM - 1), rw = threadIdx.x & (BN - 1);
    auto scales = [&](int kb0, Bytes8& vx, Bytes8& vw) {
        if constexpr (HALVES) {
            vx = second ? mx4_row_scales(W, n0 + rw, kb0) : mx4_row_scales(X, m0 + rx, kb0);
        } else {
            vx = mx4_row_scales(X, m0 + rx, kb0);
            vw = mx4_row_scales(W, n0 + rw, kb0);
        }
    };
    auto put = [&](Stage& st, uint2 vx, uint2 vw) {
        if constexpr (HALVES) {
            *reinterpret_cast<uint2*>(second ? &st.sw[rw * 2] : &st.sx[rx * 2]) = vx;
        } else {
            *reinterpret_cast<uint2*>(&st.sx[rx * 2]) = vx;
            *reinterpret_cast<uint2*>(&st.sw[rw * 2]) = vw;
        }
    };
    auto put_scales = [&](Stage& st, int kb0, Bytes8 vx, Bytes8 vw) { put(st, mx4_shift_scales(vx, W.nb, kb0), mx4_shift_scales(vw, W.nb, kb0)); };
    auto codes = [&](Stage& st, int kb0) {
        mx4_stage_codes<BM, WAVES>(X, m0, kb0, st.x);
        mx4_stage_codes<BN, WAVES>(W, n0, kb0, st.w);
    };
    auto compute = [&](const Stage& st) {
        int sx[TM], sw[TN];
#pragma unroll
        for (int j = 0; j < TM; ++j) sx[j] = (int)st.sx[(wm + j * 32 + (lane & 31)) * 2 + (lane >> 5)];
#pragma unroll
        for (int i = 0; i < TN; ++i) sw[i] = (int)st.sw[(wn + i * 32 + (lane & 31)) * 2 + (lane >> 5)];
        // the next turn's fragments are on their way while this turn's instructions run
        const uint8_t *x = st.x + wm * 128, *w = st.w + wn * 128;
        u32x4 b0[TM], a0[TN], b1[TM], a1[TN];
        mx4_turn_load<0, TM, TN>(x, w, b0, a0);
        mx4_turn_load<1, TM, TN>(x, w, b1, a1);
        mx4_turn<0, TM, TN>(b0, a0, sx, sw, acc);
        __builtin_amdgcn_sched_barrier(0);
        mx4_turn_load<2, TM, TN>(x, w, b0, a0);
        mx4_turn<1, TM, TN>(b1, a1, sx, sw, acc);
        __builtin_amdgcn_sched_barrier(0);
        mx4_turn_load<3, TM, TN>(x, w, b1, a1);
        mx4_turn<2, TM, TN>(b0, a0, sx, sw, acc);
        __builtin_amdgcn_sched_barrier(0);
        mx4_turn<3, TM, TN>(b1, a1, sx, sw, acc);
        __builtin_amdgcn_sched_barrier(0);
    };
    Bytes8 vx{0u, 0u}, vw{0u, 0u};
    const int first = blockIdx.y * span, steps = min((W.nb + 7) / 8 - first, span);
    codes(s0, first * 8);
    if (W.nb >= 8) {
        scales(first * 8, vx, vw);
        put_scales(s0, first * 8, vx, vw);
    } else {
        const uint2 sx = mx4_short_row_scales(X, m0 + rx), sw = mx4_short_row_scales(W, n0 + rw);
        put(s0, second ? sw : sx, sw);
    }
    stage_barrier();
    for (int p = 0; p < steps / 2; ++p) {
        const int kb1 = (first + 2 * p + 1) * 8, kb2 = kb1 + 8;
        scales(kb1, vx, vw);
        codes(s1, kb1);
        compute(s0);
        put_scales(s1, kb1, vx, vw);
        stage_barrier();
        scales(kb2, vx, vw);
        codes(s0, kb2);                     // behind the last step: not used
        compute(s1);
        put_scales(s0, kb2, vx, vw);
        stage_barrier();
    }
    if (steps & 1) compute(s0);
    stage_barrier();
    float* strip = reinterpret_cast<float*>(&s0) + wave * 32 * OUT_LD;
    if (part != nullptr) {
        mx4_store_tile<float, WM, WN>(strip, acc, part + (int64_t)blockIdx.y * X.rows * W.rows, W.rows, m0 + wm, n0 + wn, X.rows, W.rows, nullptr, 0);
        return;
    }
    mx4_store_tile<T, WM, WN>(strip, acc, y, ldy, m0 + wm, n0 + wn, X.rows, W.rows, bias, btype);
}

// sums of the slices of a split reduction, in order, + bias
template <typename T>
__global__ __launch_bounds__(256) void k_mx4_join(const float* __restrict__ part, int slices, int M, int N, const void* bias, int btype,
                                                  T* __restrict__ y, int64_t ldy) {
    const int64_t slots = ((int64_t)N + 3) / 4, total = (int64_t)M * slots, size = (int64_t)M * N;
    for (int64_t o = (int64_t)blockIdx.x * 256 + threadIdx.x; o < total; o += (int64_t)gridDim.x * 256) {
        const int64_t m = o / slots, n = (o - m * slots) * 4;
        float v[4], u[4];
        load_slot(part + m * N, n, N, 0.f, v);
        for (int k = 1; k < slices; ++k) {
            load_slot(part + k * size + m * N, n, N, 0.f, u);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] += u[i];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (n + i < N) y[m * ldy + n + i] = (T)(v[i] + (bias != nullptr ? load_elem(bias, btype, n + i) : 0.f));
    }
}

// ---- bias gradient: column sums of dy ----------------------------------------------------------------------------------
// A workgroup takes 32 slots of columns x 8 rows at a time, four of these under way, over a slice of the rows.
template <typename T>
__global__ __launch_bounds__(256) void k_mx4_colsum(const T* __restrict__ dy, int64_t lddy, int M, int N, float* __restrict__ part) {
    constexpr int VEC = Elem<T>::VEC, U = 4;
    __shared__ float s_sum[8][32][VEC];
    const int cl = threadIdx.x & 31, rl = threadIdx.x >> 5;
    const int64_t c0 = ((int64_t)blockIdx.x * 32 + cl) * VEC, step = (int64_t)gridDim.y * 8;
    float a[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) a[i] = 0.f;
    int64_t m = (int64_t)blockIdx.y * 8 + rl;
    if (c0 + VEC <= N)
        for (; m + (U - 1) * step < M; m += U * step) {
            Slot<T> raw[U];
#pragma unroll
            for (int u = 0; u < U; ++u) raw[u] = *reinterpret_cast<const Slot<T>*>(dy + (m + u * step) * lddy + c0);
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int i = 0; i < VEC; ++i) a[i] += (float)raw[u].v[i];
        }
    if (c0 < N)
        for (; m < M; m += step) {
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
// About four workgroups a CU, of 32 rows at least: 2048 x 8192 bf16 6.6 us (5.1 TB/s; 16 slices and one thread for each joined
// column 17 us), 1024 x 4096 4.8 us (8 rows at least 6.8).
static inline int mx4_colsum_slices(int M, int N) {
    const int64_t want = std::max<int64_t>(1, 1024 / ((N + 255ll) / 256));
    return (int)std::min<int64_t>(std::min<int64_t>(want, 256), (M + 31ll) / 32);
}

static inline int mx4_stream_grid(int64_t quads) { return (int)(quads < 256 * 16384ll ? (quads + 255) / 256 : 16384); }
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
// A reduction is split over workgroups where the tiles alone leave CUs idle: into about one workgroup a CU, of four steps at
// least, and only as far as the steps that this saves (step_us each) outweigh the join: its launch, 4 us with the host's side, and the
// partial sums, written and read at 4 TB/s.  bf16 x: 64 x 4096 x 4096 17 us, whole 31 us (gradient 18 and 40), 64 x 4096 x 2048 13 and 17;
// 512 x 2048 x 2048 would be 23 us in four slices, whole it is 18.  Both in 4 bits: 257 x 1000 x 8192 11 us, whole 15; x 4080 9.5 and 9.0.
// Returns the number of slices and the steps of each.
static inline int mx4_split(int64_t tiles, int steps, double step_us, int M, int N, int& span) {
    const int64_t want = tiles < 192 ? 256 / (tiles > 0 ? tiles : 1) : 1;
    int slices = (int)std::max<int64_t>(1, std::min<int64_t>(want, steps / 4));
    while (slices > 1 && (steps - (steps + slices - 1) / slices) * step_us <= 4.0 + 2.0 * slices * M * N * sizeof(float) / 4e6) slices /= 2;
    span = (steps + slices - 1) / slices;
    return (steps + span - 1) / span;
}
// one step of a tile's workgroup, from products that were not split: 128 of the reduction for bf16 rows, 64 for the parts of the wider types
static inline double mx4_step_us(int dtype) { return dtype == DRM_BF16 ? 0.85 : dtype == DRM_F16 ? 1.1 : 1.6; }
constexpr double MX4_PRODUCT_STEP_US = 0.4;
static inline int64_t mx4_tiles(int M, int N, int b) { return (int64_t)((M + b - 1) / b) * ((N + b - 1) / b); }
static inline size_t mx4_part_bytes(int slices, int M, int N) { return slices > 1 ? (size_t)slices * M * N * sizeof(float) : 0; }
static inline int mx4_step_of(int dtype) { return dtype == DRM_BF16 ? 128 : 64; }

// Large products: bf16 rows whose 16-byte chunks are aligned and whole go to LDS by direct loads with 128 of the reduction per step
// (side by side: 1024 x 4096 x 4096 45.6 us, through registers 50.0; 2048 x 8192 x 4096 153 and 166), in three stages where a row's
// scales are whole dwords (two: 46.2 and 156 us); through registers the parts of wider types leave room for 64.
template <bool GRAD, typename T>
static void mx4_launch_tile(const T* x, int64_t ldx, const Mx4& W, const void* bias, int btype, T* y, int64_t ldy, int M, int N, int K,
                            float* part, hipStream_t s) {
    const int tm = (M + 127) / 128, tn = (N + 127) / 128;
    constexpr int BK = Parts<T>::N == 1 ? 128 : 64;
    int span = 0;
    const int slices = mx4_split((int64_t)tm * tn, (K + BK - 1) / BK, mx4_step_us(Elem<T>::ID), M, N, span);
    if (slices == 1) part = nullptr;
    const dim3 grid(tm * tn, slices);
    auto go = [&](auto direct, auto ring) {
        constexpr bool DIRECT = decltype(direct)::value, RING = decltype(ring)::value;
        k_mx4_tile<T, BK, DIRECT, GRAD, RING><<<grid, TILE_THREADS, 0, s>>>(x, ldx, W, bias, btype, y, ldy, M, N, K, tm, tn, part, span * BK);
    };
    bool done = false;
    if constexpr (Parts<T>::N == 1) {
        if (aligned16(x) && ldx % 8 == 0 && K % 8 == 0 && ldx <= (1 << 22)) {
            if constexpr (!GRAD) {
                if (W.nb % 4 == 0 && ((uintptr_t)W.scales & 3) == 0) { go(std::true_type{}, std::true_type{}); done = true; }
            }
            if (!done) { go(std::true_type{}, std::false_type{}); done = true; }
        }
    }
    if (!done) go(std::false_type{}, std::false_type{});
    if (part != nullptr) k_mx4_join<T><<<mx4_stream_grid((int64_t)M * ((N + 3) / 4)), 256, 0, s>>>(part, slices, M, N, bias, btype, y, ldy);
}
// Few rows: as many weight tiles per wave as leave about one workgroup a CU (x is read once per workgroup): bf16 16 x 12288 x 4096
// with 1 / 2 / 4 tiles 11.4 / 11.5 / 9.3 us, 16 x 8192 x 8192 13.9 / 10.7 / 15.2 us, 16 x 4096 x 4096 5.1 / 6.1 / 8.8 us.  Eight
// waves where two stages of their passes fit the LDS, else four (1 x 4096 x 4096 4.6 us, with four 5.1).  Up to 32 rows: 32 x 12288 x
// 4096 12 us, the tiles above 21 us (16 rows 9.3 and 20 us, fp32 32 x 4096 x 4096 21.5 and 23.6 us); 33 rows would take three row
// tiles and their tile kernel takes 15 us at 4096 x 4096.
constexpr int MX4_FEW_ROWS = 32;
template <typename T, int MT>
static void mx4_launch_rows_mt(const T* x, int64_t ldx, const Mx4& W, const void* bias, int btype, T* y, int64_t ldy, int M, int N, int K, hipStream_t s) {
    constexpr int EPC = 16 / sizeof(T), NW = MT * sizeof(T) <= 2 ? 8 : 4, MAX_NT = MT * sizeof(T) <= 4 ? 4 : 2;
    if (!aligned16(x) || ldx % EPC != 0 || K % 8 != 0) {
        k_mx4_rows_any<T, MT, 8><<<(N + 15) / 16, 512, 0, s>>>(x, ldx, W, bias, btype, y, ldy, M, K);
        return;
    }
    auto go = [&](auto nt) {
        constexpr int NT = decltype(nt)::value;
        k_mx4_rows<T, MT, NT, NW><<<(N + 16 * NT - 1) / (16 * NT), NW * 64, 0, s>>>(x, ldx, W, bias, btype, y, ldy, M, K);
    };
    if constexpr (MAX_NT == 4) {
        if (N >= 64 * 192) { go(std::integral_constant<int, 4>{}); return; }
    }
    if (N >= 32 * 192) go(std::integral_constant<int, 2>{});
    else go(std::integral_constant<int, 1>{});
}
template <typename T>
static void mx4_launch_rows(const T* x, int64_t ldx, const Mx4& W, const void* bias, int btype, T* y, int64_t ldy, int M, int N, int K, hipStream_t s) {
    // (as many rows of the weight as one launch of 16 rows for 512 threads takes)
    const int64_t most = launch_limit(512) * 16;
    for (int64_t n = 0; n < N; n += most) {
        const int rows = (int)std::min<int64_t>(N - n, most);
        const Mx4 P{W.codes + n * W.nb * 16, W.scales + n * W.nb, rows, W.nb};
        const void* b = bias != nullptr ? (const char*)bias + n * elem_bytes(btype) : nullptr;
        if (M <= 16) mx4_launch_rows_mt<T, 1>(x, ldx, P, b, btype, y + n, ldy, M, rows, K, s);
        else mx4_launch_rows_mt<T, 2>(x, ldx, P, b, btype, y + n, ldy, M, rows, K, s);
    }
}

static int mx4_check_tiles(const char* what, int M, int N, int K, int tile) {
    DRM_REQUIRE(K <= (1 << 22), DRM_ENOTSUP, "%s: a row of %d elements (at most 4194304)", what, K);
    DRM_REQUIRE(M <= 65535 * 128, DRM_ENOTSUP, "%s: M=%d rows (at most %d)", what, M, 65535 * 128);
    // (of 512 threads, and a launch takes fewer than 2^32 along an axis; 0: no tiles)
    DRM_REQUIRE(tile == 0 || mx4_tiles(M, N, tile) < 1 << 23, DRM_ENOTSUP, "%s: M=%d N=%d: too many tiles", what, M, N);
    return DRM_OK;
}

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
        k_mx4_dequantize<T><<<mx4_stream_grid(rows * nb * (32 / Elem<T>::VEC)), 256, 0, s>>>(codes, scales, rows, K, nb, (T*)y, ldy);
        DRM_LAUNCH_CHECK();
        return DRM_OK;
    });
}

// The largest tile (fewest bytes through LDS per product) whose tiles still give most CUs one.  Tiles of 256 / 128 / 64: 4096^3 45 / 58 /
// 85 us, 2048 x 6144 x 4096 (192 tiles of 256) 40 / 46 / 69 us, 1024 x 4096 x 4096 (256 of 128) 40 / 20 / 27 us, 257 x 1000 x 4080 20 / 12 /
// 10 us.
static int mx4_product_tile(int M, int N) { return mx4_tiles(M, N, 256) >= 192 ? 256 : mx4_tiles(M, N, 128) >= 192 ? 128 : 64; }

static int mx4_check_workspace(const char* what, const void* ws, size_t have, size_t need) {
    DRM_REQUIRE(need == 0 || (ws && have >= need && aligned16(ws)), DRM_EINVAL, "%s: workspace of %zu bytes, %zu needed (16-byte aligned)", what,
                ws ? have : (size_t)0, need);
    return DRM_OK;
}

extern "C" size_t drm_mx4_linear_workspace_bytes(int32_t dtype, int32_t M, int32_t N, int32_t K) {
    if (!elem_ok(dtype) || M <= MX4_FEW_ROWS || N < 1 || K < 1) return 0;
    int span = 0;
    const int bk = mx4_step_of(dtype);
    return mx4_part_bytes(mx4_split(mx4_tiles(M, N, 128), (K - 1) / bk + 1, mx4_step_us(dtype), M, N, span), M, N);
}
extern "C" size_t drm_mx4_linear_dgrad_workspace_bytes(int32_t dtype, int32_t M, int32_t N, int32_t K) {
    if (!elem_ok(dtype) || M < 1 || N < 1 || K < 1) return 0;
    int span = 0;
    const int bk = mx4_step_of(dtype);
    return mx4_part_bytes(mx4_split(mx4_tiles(M, K, 128), (N - 1) / bk + 1, mx4_step_us(dtype), M, K, span), M, K);
}
extern "C" size_t drm_mx4_product_workspace_bytes(int32_t M, int32_t N, int32_t K) {
    if (M < 1 || N < 1 || K < 1) return 0;
    int span = 0;
    return mx4_part_bytes(mx4_split(mx4_tiles(M, N, mx4_product_tile(M, N)), (mx4_blocks(K) + 7) / 8, MX4_PRODUCT_STEP_US, M, N, span), M, N);
}

extern "C" int drm_mx4_linear(const void* x, int64_t ldx, int32_t dtype, const uint8_t* codes, const uint8_t* scales, const void* bias,
                              int32_t bias_dtype, void* y, int64_t ldy, int32_t M, int32_t N, int32_t K, void* workspace,
                              size_t workspace_bytes, drm_stream_t stream) {
    if (M == 0 && N >= 1 && K >= 1) return DRM_OK;
    if (int rc = mx4_check(__func__, codes, scales, N, K)) return rc;
    if (int rc = mx4_check_product(__func__, x, ldx, dtype, K, bias, bias_dtype, y, ldy, N, M)) return rc;
    if (int rc = mx4_check_tiles(__func__, M, N, K, M <= MX4_FEW_ROWS ? 0 : 128)) return rc;
    if (int rc = mx4_check_workspace(__func__, workspace, workspace_bytes, drm_mx4_linear_workspace_bytes(dtype, M, N, K))) return rc;
    hipStream_t s = (hipStream_t)stream;
    const Mx4 W{codes, scales, N, mx4_blocks(K)};
    ProfScope ps(M <= MX4_FEW_ROWS ? PC_LINEAR : PC_LINEAR_BIG, s, 2.0 * M * N * K, ((double)M * K + (double)M * N) * elem_bytes(dtype) + (double)N * W.nb * 17);
    return with_elem(dtype, [&](auto tag) -> int {
        using T = decltype(tag);
        if (M <= MX4_FEW_ROWS) mx4_launch_rows<T>((const T*)x, ldx, W, bias, bias_dtype, (T*)y, ldy, M, N, K, s);
        else mx4_launch_tile<false, T>((const T*)x, ldx, W, bias, bias_dtype, (T*)y, ldy, M, N, K, (float*)workspace, s);
        DRM_LAUNCH_CHECK();
        return DRM_OK;
    });
}

extern "C" int drm_mx4_linear_dgrad(const void* dy, int64_t lddy, int32_t dtype, const uint8_t* codes, const uint8_t* scales, void* dx,
                                    int64_t lddx, int32_t M, int32_t N, int32_t K, void* workspace, size_t workspace_bytes,
                                    drm_stream_t stream) {
    if (M == 0 && N >= 1 && K >= 1) return DRM_OK;
    if (int rc = mx4_check(__func__, codes, scales, N, K)) return rc;
    if (int rc = mx4_check_product(__func__, dy, lddy, dtype, N, nullptr, 0, dx, lddx, K, M)) return rc;
    if (int rc = mx4_check_tiles(__func__, M, K, K, 128)) return rc;
    DRM_REQUIRE(N >= 1 && N <= (1 << 30), DRM_EINVAL, "N=%d", N);
    if (int rc = mx4_check_workspace(__func__, workspace, workspace_bytes, drm_mx4_linear_dgrad_workspace_bytes(dtype, M, N, K))) return rc;
    hipStream_t s = (hipStream_t)stream;
    const Mx4 W{codes, scales, N, mx4_blocks(K)};
    ProfScope ps(PC_LINEAR_BIG, s, 2.0 * M * N * K, ((double)M * K + (double)M * N) * elem_bytes(dtype) + (double)N * W.nb * 17);
    return with_elem(dtype, [&](auto tag) -> int {
        using T = decltype(tag);
        mx4_launch_tile<true, T>((const T*)dy, lddy, W, nullptr, 0, (T*)dx, lddx, M, K, N, (float*)workspace, s);
        DRM_LAUNCH_CHECK();
        return DRM_OK;
    });
}

extern "C" int drm_mx4_product(const uint8_t* x_codes, const uint8_t* x_scales, const uint8_t* w_codes, const uint8_t* w_scales,
                               const void* bias, int32_t bias_dtype, void* y, int64_t ldy, int32_t y_dtype, int32_t M, int32_t N,
                               int32_t K, void* workspace, size_t workspace_bytes, drm_stream_t stream) {
    if (M == 0 && N >= 1 && K >= 1) return DRM_OK;
    if (int rc = mx4_check(__func__, x_codes, x_scales, M, K)) return rc;
    if (int rc = mx4_check(__func__, w_codes, w_scales, N, K)) return rc;
    if (int rc = mx4_check_product(__func__, x_codes, K, y_dtype, K, bias, bias_dtype, y, ldy, N, M)) return rc;
    if (int rc = mx4_check_tiles(__func__, M, N, K, mx4_product_tile(M, N))) return rc;
    if (int rc = mx4_check_workspace(__func__, workspace, workspace_bytes, drm_mx4_product_workspace_bytes(M, N, K))) return rc;
    hipStream_t s = (hipStream_t)stream;
    const Mx4 X{x_codes, x_scales, M, mx4_blocks(K)}, W{w_codes, w_scales, N, mx4_blocks(K)};
    ProfScope ps(PC_LINEAR_BIG, s, 2.0 * M * N * K, (double)M * N * elem_bytes(y_dtype) + ((double)M + N) * W.nb * 17);
    return with_elem(y_dtype, [&](auto tag) -> int {
        using T = decltype(tag);
        const int b = mx4_product_tile(M, N), tm = (M + b - 1) / b, tn = (N + b - 1) / b;
        int span = 0;
        const int slices = mx4_split((int64_t)tm * tn, (W.nb + 7) / 8, MX4_PRODUCT_STEP_US, M, N, span);
        float* part = slices > 1 ? (float*)workspace : nullptr;
        const dim3 grid(tm * tn, slices);
        if (b == 256) k_mx4_product<T, 256, 256, 128, 64><<<grid, 512, 0, s>>>(X, W, bias, bias_dtype, (T*)y, ldy, tm, tn, part, span);
        else if (b == 128) k_mx4_product<T, 128, 128, 64, 32><<<grid, 512, 0, s>>>(X, W, bias, bias_dtype, (T*)y, ldy, tm, tn, part, span);
        else k_mx4_product<T, 64, 64, 32, 32><<<grid, 256, 0, s>>>(X, W, bias, bias_dtype, (T*)y, ldy, tm, tn, part, span);
        if (part != nullptr) k_mx4_join<T><<<mx4_stream_grid((int64_t)M * ((N + 3) / 4)), 256, 0, s>>>(part, slices, M, N, bias, bias_dtype, (T*)y, ldy);
        DRM_LAUNCH_CHECK();
        return DRM_OK;
    });
}

extern "C" size_t drm_mx4_bias_grad_workspace_bytes(int32_t M, int32_t N) {
    if (M < 1 || N < 1) return 0;
    return (size_t)mx4_colsum_slices(M, N) * N * sizeof(float);
}

extern "C" int drm_mx4_bias_grad(const void* dy, int64_t lddy, int32_t dtype, void* db, int32_t db_dtype, int32_t M, int32_t N,
                                 void* workspace, size_t workspace_bytes, drm_stream_t stream) {
    DRM_REQUIRE(dy && db, DRM_EINVAL, "null pointer");
    DRM_REQUIRE(elem_ok(dtype) && elem_ok(db_dtype), DRM_ENOTSUP, "element types %d / %d (fp32, bf16 or fp16)", dtype, db_dtype);
    DRM_REQUIRE(M >= 1 && N >= 1 && N <= INT_MAX - 512 && lddy >= N, DRM_EINVAL, "M=%d N=%d row stride %lld", M, N, (long long)lddy);
    const size_t need = drm_mx4_bias_grad_workspace_bytes(M, N);
    DRM_REQUIRE(workspace && workspace_bytes >= need, DRM_EINVAL, "workspace of %zu bytes, %zu needed", workspace ? workspace_bytes : (size_t)0, need);
    hipStream_t s = (hipStream_t)stream;
    const int slices = mx4_colsum_slices(M, N);
    ProfScope ps(PC_ELEMENTWISE, s, (double)M * N, (double)M * N * elem_bytes(dtype));
    const int rc = with_elem(dtype, [&](auto tag) -> int {
        using T = decltype(tag);
        constexpr int COLS = 32 * Elem<T>::VEC;
        k_mx4_colsum<T><<<dim3((N + COLS - 1) / COLS, slices), 256, 0, s>>>((const T*)dy, lddy, M, N, (float*)workspace);
        DRM_LAUNCH_CHECK();
        return DRM_OK;
    });
    if (rc != DRM_OK) return rc;
    join_columns((const float*)workspace, slices, N, N, db_dtype, db, nullptr, s);
    DRM_LAUNCH_CHECK();
    return DRM_OK;
}
