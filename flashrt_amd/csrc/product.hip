// Products of the sorted rows with their experts' matrices, and both gradients, on the matrix cores: operands of 32 or 16 bits, sums in fp32.
//
//   product   out[r] = w_g a(r)          contracted over C, both operands' rows
//   grad      da[r] = w_g^T dout[r]      contracted over N: w's columns
//   wgrad     dw_g = sum_r dout[r] a(r)^T   contracted over the group's rows: columns of both
// r in [bounds[g], bounds[g + 1]); a(r) is row r, or row rows[r]. In all three an output tile is X Y^T with X the operand along the output's
// rows and Y the one along its columns ("features"). Three kernels, by alignment and size: tiles through direct loads into LDS (whole, aligned
// rows of 16 bits), tiles through registers (any rows, and 32 bits), and rows straight into the matrix instructions (few rows).
#include "common.hpp"
#include "groups.hpp"
#include "lds_dma.hpp"
#include "mx8.hpp"

#include <algorithm>
#include <type_traits>

#include "../../include/flashrt_moe.h"
#include "product.hpp"

namespace frt {

typedef uint32_t u4e4_t __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u4e2_t __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u2e2_t __attribute__((ext_vector_type(2), aligned(2)));
typedef float f4_t __attribute__((ext_vector_type(4)));
typedef float f16_t __attribute__((ext_vector_type(16)));
typedef short s4_t __attribute__((ext_vector_type(4)));

enum Mode { kProduct, kGrad, kWgrad };

// (lambdas of several calls: left to itself the compiler calls the largest, and what they capture goes to memory)
#define INLINE __attribute__((always_inline))

// 16 bytes of an operand's row: what a lane gives the matrix instructions for one step
template <typename T>
struct Chunk {
    static constexpr int V = 16 / sizeof(T);
    typedef T Vec __attribute__((ext_vector_type(V)));
    typedef std::conditional_t<sizeof(T) == 4, u4e4_t, u4e2_t> Raw;   // at the element's own alignment
};
template <typename T>
using Vec = typename Chunk<T>::Vec;

// acc += y x^T over the V values of each lane half: 32 features x 32 rows. Lane l gives feature and row l % 32, values of half l / 32.
__device__ __forceinline__ f16_t mma(Vec<_Float16> y, Vec<_Float16> x, f16_t acc) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(y, x, acc, 0, 0, 0); }
__device__ __forceinline__ f16_t mma(Vec<__bf16> y, Vec<__bf16> x, f16_t acc) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(y, x, acc, 0, 0, 0); }
__device__ __forceinline__ f16_t mma(Vec<float> y, Vec<float> x, f16_t acc) {
#pragma unroll
    for (int i = 0; i < 4; ++i) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(y[i], x[i], acc, 0, 0, 0);
    return acc;
}

// Four 16-bit values of sixteen columns. (Without __restrict, here and at the direct loads, the compiler has these reads wait for every direct
// load under way, which might write what they read; the waits in the code see to that.)
__device__ __forceinline__ s4_t read_tr(const uint8_t* __restrict s) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4_t*)const_cast<uint8_t*>(s));
}

// A stage of an operand in LDS: W rows (or columns) of KB chunks of contracted values, of which step t takes 2 t and 2 t + 1 (one per lane
// half). ROW: [W][KB chunks], chunk c of row r at c ^ (r / (16 / KB) % KB), so that the sixteen rows of a read phase take sixteen different
// columns of the banks. COL: [KB V][W], the contracted values apart: chunks of 16 bits are read by the transposing LDS read, four
// values of sixteen columns at a time (a lane's address is a quarter of one row's 32 bytes), 32-bit ones value by value; 32-byte
// blocks of rows that a read takes together lie in different banks.
template <typename T, int W, bool COL, int KB>
struct Stage {
    static constexpr int V = Chunk<T>::V, BK = KB * V, bytes = W * KB * 16;
    static constexpr int row_b = COL ? W * int(sizeof(T)) : KB * 16, PR = row_b / 16;   // bytes and pieces of a stored row
    static constexpr int Q = row_b < 256 ? 256 / row_b : 1;
    static __device__ __forceinline__ int swizzle(int r) { return COL ? ((r / Q & 3) << 2) & (PR - 1) : r / Q % KB; }
    static __device__ __forceinline__ int piece(int r, int p) { return r * row_b + ((p ^ swizzle(r)) << 4); }
    // The lane's chunk of step t of rows (columns) w0 .. w0 + 31
    static __device__ __forceinline__ Vec<T> read(const uint8_t* s, int w0, int t) {
        const int lane = threadIdx.x & 63, j = lane & 31, c = 2 * t + (lane >> 5);
        if constexpr (!COL) {
            return *reinterpret_cast<const Vec<T>*>(s + piece(w0 + j, c));
        } else if constexpr (sizeof(T) == 4) {
            Vec<T> v;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int k = c * V + i, b = (w0 + j) * 4;
                v[i] = *reinterpret_cast<const float*>(s + piece(k, b >> 4) + (b & 15));
            }
            return v;
        } else {
            const int b = (w0 + (lane & 16) + (lane & 3) * 4) * 2, k = c * V + ((lane & 15) >> 2);
            const s4_t lo = read_tr(s + piece(k, b >> 4) + (b & 15));
            const s4_t hi = read_tr(s + piece(k + 4, b >> 4) + (b & 15));
            return __builtin_bit_cast(Vec<T>, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        }
    }
};

// The chunk of a row of n values that begins at c, zeros past the end (and of no row)
template <typename T>
__device__ __forceinline__ Vec<T> load_chunk(const T* row, int64_t c, int64_t n) {
    constexpr int V = Chunk<T>::V;
    Vec<T> v = {};
    if (!row || c >= n) return v;
    if (c + V <= n) return __builtin_bit_cast(Vec<T>, *reinterpret_cast<const typename Chunk<T>::Raw*>(row + c));
    for (int i = 0; i < V; ++i)
        if (c + i < n) v[i] = row[c + i];
    return v;
}
// The same of a row in 8 bits, rounded to T
template <typename T>
__device__ __forceinline__ Vec<T> load_chunk8(const uint8_t* codes, const uint8_t* scales, int64_t row, int64_t c, int64_t n) {
    constexpr int V = Chunk<T>::V;
    Vec<T> v = {};
    if (row < 0 || c >= n) return v;   // (n is a multiple of 32)
    const uint32_t* const q = reinterpret_cast<const uint32_t*>(codes + row * n + c);
    const auto f = mx8_values(q[0], V == 8 ? q[V / 4 - 1] : 0, mx8_scale(scales[row * (n / 32) + c / 32]));
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = T(f[i]);
    return v;
}

// Four adjacent results of a row from column c, of which `left` are inside
template <typename O>
__device__ __forceinline__ void store4(O* o, f4_t v, int left, bool add) {
    typedef O v4 __attribute__((ext_vector_type(4)));
    typedef std::conditional_t<sizeof(O) == 4, u4e4_t, u2e2_t> Raw;
    if (left >= 4) {
        if (add) v += __builtin_convertvector(__builtin_bit_cast(v4, *reinterpret_cast<const Raw*>(o)), f4_t);
        *reinterpret_cast<Raw*>(o) = __builtin_bit_cast(Raw, __builtin_convertvector(v, v4));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < left) o[i] = O(add ? v[i] + float(o[i]) : v[i]);
    }
}
__device__ __forceinline__ void store4(const ProductArgs& p, int64_t at, f4_t v, int left) {
    if (p.out_type == FRT_GGML_F32)
        store4(static_cast<float*>(p.out) + at, v, left, p.add);
    else if (p.out_type == FRT_GGML_F16)
        store4(static_cast<_Float16*>(p.out) + at, v, left, p.add);
    else
        store4(static_cast<__bf16*>(p.out) + at, v, left, p.add);
}

// Rows at any distance and alignment, and calls of few tiles: a tile of BM rows x BN features by KS times WM x WN waves, each share of which takes
// every KS-th stage of the summed values into its own LDS, the next one's operands in registers while this one is multiplied; the shares' sums are
// added through LDS in their order. What hides the loads' latency is the other shares and the other workgroups of the CU. 1542 rows of 128 experts (N
// 1021, C 1019, fp16, 267 MB of weights) 62 us (73 from memory), about the time of the other kernels at C 1024; 16384 rows 136 us, 250 TFLOP/s; fp32
// (8192 rows, N 2048, C 2048) 119 TFLOP/s of the library's 153 at 8192^3. Whole stages without the checks of single pieces gave nothing. (Two
// workgroups of 128 x 128 to a CU: fp32 with 8-bit rows spills two registers.)
template <typename T, Mode MODE, bool EIGHT, int BM, int BN, int WM, int WN, int KS>
__global__ void __launch_bounds__(64 * WM * WN * KS, BM == 128 ? 4 : 1) k_product_any(ProductArgs p, int nx, int ny, FastDiv divx, FastDiv divy) {
    constexpr int NT = 64 * WM * WN, V = Chunk<T>::V, FM = BM / WM / 32, FN = BN / WN / 32;
    constexpr bool XCOL = MODE == kWgrad, YCOL = MODE != kProduct;
    using SX = Stage<T, BM, XCOL, 8>;
    using SY = Stage<T, BN, YCOL, 8>;
    constexpr int PX = BM * 8 / NT, PY = BN * 8 / NT, BK = SX::BK;
    static_assert(BM * 8 % NT == 0 && BN * 8 % NT == 0, "whole pieces per thread");
    extern __shared__ __align__(16) uint8_t smem[];
    const int kg = __builtin_amdgcn_readfirstlane(threadIdx.x / NT), tid = threadIdx.x % NT;   // the share of the stages, and the thread in it
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    uint8_t* const s_x = smem + kg * (SX::bytes + SY::bytes);
    uint8_t* const s_y = s_x + SX::bytes;
    int* const s_row = reinterpret_cast<int*>(smem + KS * (SX::bytes + SY::bytes));   // [BM]
    const uint32_t unit = wide_block(), outer = divy(unit);
    const int y0 = int(unit - outer * ny) * BN;
    int g, x0, xn, K, k_first = 0;   // the tile's group, first row and rows, and the contracted values (from k_first on)
    if constexpr (MODE == kWgrad) {
        g = int(divx(outer));
        x0 = int(outer - uint32_t(g) * nx) * BM;
        xn = min(BM, p.N - x0);
        if (g >= p.E) return;
        k_first = p.bounds ? min(max(p.bounds[g], 0), p.M) : 0;
        K = (p.bounds ? min(max(p.bounds[g + 1], 0), p.M) : p.M) - k_first;
        if (K <= 0 && p.add) return;
    } else {
        const RowTile t = find_tile<BM>(p.bounds, p.E, p.M, [&](int total) { return int(outer) < total ? int(outer) : -1; });
        if (t.rows == 0) return;
        g = t.g;
        x0 = t.row0;
        xn = t.rows;
        K = MODE == kProduct ? p.C : p.N;
        for (int i = threadIdx.x; i < BM; i += NT * KS) {
            const int r = x0 + min(i, xn - 1);
            const int a = p.rows ? p.rows[r] : r;
            s_row[i] = i < xn && unsigned(a) < unsigned(p.a_rows) ? a : -1;
        }
        __syncthreads();
    }
    const int features = MODE == kProduct ? p.N : p.C;
    const T* const x = static_cast<const T*>(p.x);
    const T* const y = static_cast<const T*>(p.y) + (MODE == kWgrad ? 0 : int64_t(g) * p.N * p.C);
    Vec<T> rx[PX], ry[PY];
    auto load = [&](int k0) {
#pragma unroll
        for (int i = 0; i < PX; ++i) {
            const int q = i * NT + tid, r = q / SX::PR, c = q % SX::PR;
            if constexpr (XCOL) {
                const int64_t k = int64_t(k0) + r;
                rx[i] = load_chunk(k < K ? x + (k_first + k) * p.ldx : nullptr, int64_t(x0) + c * V, p.N);
            } else {
                const int a = s_row[r];
                rx[i] = load_chunk(a < 0 ? nullptr : x + a * p.ldx, int64_t(k0) + c * V, K);
            }
        }
#pragma unroll
        for (int i = 0; i < PY; ++i) {
            const int q = i * NT + tid, r = q / SY::PR, c = q % SY::PR;
            if constexpr (MODE == kProduct) {
                ry[i] = load_chunk(y0 + r < features ? y + int64_t(y0 + r) * K : nullptr, int64_t(k0) + c * V, K);
            } else if constexpr (MODE == kGrad) {
                const int64_t k = int64_t(k0) + r;
                ry[i] = load_chunk(k < K ? y + k * p.C : nullptr, int64_t(y0) + c * V, p.C);
            } else {
                const int64_t k = int64_t(k0) + r;
                int64_t a = -1;
                if (k < K) {
                    a = p.rows ? p.rows[k_first + k] : k_first + k;
                    if (a >= p.a_rows) a = -1;
                }
                if constexpr (EIGHT)
                    ry[i] = load_chunk8<T>(static_cast<const uint8_t*>(p.y), p.scales, a, int64_t(y0) + c * V, p.C);
                else
                    ry[i] = load_chunk(a < 0 ? nullptr : y + a * p.ldy, int64_t(y0) + c * V, p.C);
            }
        }
    };
    const int wm = wave / WN * FM * 32, wn = wave % WN * FN * 32;
    // Sums of fp32 operands are formed in two steps, of kPart stages (256 values) and of these, so that their error grows with the
    // two lengths and not with their product; 16-bit ones' add sixteen products at a time as it is.
    constexpr bool PARTS = sizeof(T) == 4;
    constexpr int kPart = 8;
    f16_t acc[FM][FN], sum[FM][FN];
    auto clear = [&](f16_t (&v)[FM][FN]) INLINE {
#pragma unroll
        for (int m = 0; m < FM; ++m)
#pragma unroll
            for (int f = 0; f < FN; ++f)
#pragma unroll
                for (int i = 0; i < 16; ++i) v[m][f][i] = 0.0f;
    };
    auto add = [&](f16_t (&v)[FM][FN], const f16_t (&w)[FM][FN]) INLINE {
#pragma unroll
        for (int m = 0; m < FM; ++m)
#pragma unroll
            for (int f = 0; f < FN; ++f) v[m][f] += w[m][f];
    };
    clear(acc);
    clear(sum);
    const int step = BK * KS;   // (a share past the values multiplies zeros)
    int part = 0;
    if (K > 0) load(kg * BK);
    for (int k0 = kg * BK; k0 - kg * BK < K; k0 += step) {
        __syncthreads();   // every wave has read the stage before
#pragma unroll
        for (int i = 0; i < PX; ++i) {
            const int q = i * NT + tid;
            *reinterpret_cast<Vec<T>*>(s_x + SX::piece(q / SX::PR, q % SX::PR)) = rx[i];
        }
#pragma unroll
        for (int i = 0; i < PY; ++i) {
            const int q = i * NT + tid;
            *reinterpret_cast<Vec<T>*>(s_y + SY::piece(q / SY::PR, q % SY::PR)) = ry[i];
        }
        __syncthreads();
        if (K - (k0 - kg * BK) > step) load(k0 + step);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            Vec<T> b[FN];
#pragma unroll
            for (int f = 0; f < FN; ++f) b[f] = SY::read(s_y, wn + 32 * f, t);
#pragma unroll
            for (int m = 0; m < FM; ++m) {
                const Vec<T> a = SX::read(s_x, wm + 32 * m, t);
#pragma unroll
                for (int f = 0; f < FN; ++f) acc[m][f] = mma(b[f], a, acc[m][f]);
            }
        }
        if (PARTS && ++part == kPart) {
            part = 0;
            add(sum, acc);
            clear(acc);
        }
    }
    if constexpr (PARTS) add(acc, sum);
    if constexpr (KS > 1) {   // the shares' sums, in their order
        static_assert(BM * BN * 4 <= SX::bytes + SY::bytes, "a share's sums in its stage");
        __syncthreads();
        f16_t* const mine = reinterpret_cast<f16_t*>(s_x);
#pragma unroll
        for (int m = 0; m < FM; ++m)
#pragma unroll
            for (int f = 0; f < FN; ++f) mine[(m * FN + f) * NT + tid] = acc[m][f];
        __syncthreads();
        if (kg != 0) return;
#pragma unroll
        for (int j = 1; j < KS; ++j)
#pragma unroll
            for (int m = 0; m < FM; ++m)
#pragma unroll
                for (int f = 0; f < FN; ++f)
                    acc[m][f] += reinterpret_cast<const f16_t*>(smem + j * (SX::bytes + SY::bytes))[(m * FN + f) * NT + tid];
    }
    // Lane l's value i of a fragment: feature 8 (i / 4) + 4 (l / 32) + i % 4, row l % 32
    const int64_t out0 = MODE == kWgrad ? int64_t(g) * p.N * p.C : 0;
#pragma unroll
    for (int m = 0; m < FM; ++m) {
        const int r = wm + 32 * m + (lane & 31);
        if (r >= xn) continue;
        const int64_t o = out0 + (int64_t(x0) + r) * p.ldout;
#pragma unroll
        for (int f = 0; f < FN; ++f)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int c = y0 + wn + 32 * f + 8 * q + 4 * (lane >> 5);
                if (c < features) store4(p, o + c, f4_t{acc[m][f][4 * q], acc[m][f][4 * q + 1], acc[m][f][4 * q + 2], acc[m][f][4 * q + 3]}, features - c);
            }
    }
}

template <typename T, Mode MODE, bool EIGHT, int BM, int BN, int WM, int WN, int KS>
static int any_go(const char* what, const ProductArgs& p, hipStream_t stream) {
    const int features = MODE == kProduct ? p.N : p.C, ny = (features + BN - 1) / BN, nx = (p.N + BM - 1) / BM;
    const int64_t units = (MODE == kWgrad ? int64_t(p.E) * nx : tiles_at_most(p.M, p.E, BM, p.bounds != nullptr)) * ny;
    constexpr int smem = KS * (BM + BN) * 128 + BM * 4;
    static_assert(smem <= 160 * 1024 && 64 * WM * WN * KS <= 1024, "LDS of a CU, threads of a workgroup");
    if (units > 0x7ffff000) return set_error(kErrShape, "%s: M=%d N=%d C=%d E=%d", what, p.M, p.N, p.C, p.E);
    if constexpr (smem > 64 * 1024)
        FRT_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(&k_product_any<T, MODE, EIGHT, BM, BN, WM, WN, KS>),
                                    hipFuncAttributeMaxDynamicSharedMemorySize, smem));
    launch_timed(what, k_product_any<T, MODE, EIGHT, BM, BN, WM, WN, KS>, wide_grid(uint32_t(units), 64 * WM * WN * KS), dim3(64 * WM * WN * KS), smem,
                 stream, p, nx, ny, FastDiv(uint32_t(nx)), FastDiv(uint32_t(ny)));
    FRT_LAUNCHED(what);
    return kOk;
}
// A group's rows, and the tiles of BM x BN that a call has, were the rows spread evenly over the groups that can have some
static int64_t even_rows(const ProductArgs& p) { return p.M / (p.bounds ? std::min(p.E, std::max(p.M, 1)) : 1); }
template <Mode MODE>
static int64_t even_tiles(const ProductArgs& p, int64_t BM, int64_t BN) {
    const int64_t groups = p.bounds ? std::min(p.E, std::max(p.M, 1)) : 1;
    return (MODE == kWgrad ? p.E * ((p.N + BM - 1) / BM) : (even_rows(p) + BM - 1) / BM * groups) * (((MODE == kProduct ? p.N : p.C) + BN - 1) / BN);
}
// Up to as many tiles of 64 x 64 as CUs leave CUs or their matrix cores idle, so the summed values are shared out over a workgroup's waves,
// the more of them the fewer tiles there are; many tiles are read the less often the larger they are.
// us, 32 x 32 over 16 shares / 64 x 64 over 4 / over 2 / undivided / 128 x 128, weights from memory:
//   16-bit product, N and C odd: 128 experts of 4 rows (N 1021, C 1019, 266 MB) 174 / 78 / 64 / 66 / 63, of 12 rows 191 / 81 / 67 / 70 / 67; one group of
//   4096 rows (C 2047, N 2048) 524 / 141 / 110 / 114 / 74, of 1024 rows (N 1024) 64 / 24 / 27 / 35 / 47
//   weights' gradient (N 511, C 509) of one group of 8192 rows 77 / 132 / 198 / 348 / 546; of 2048 rows each, four groups 87 / 38 / 57 / 101 / 153,
//   sixteen 328 / 142 / 170 / 174 / 171, of 1024 rows, 32 groups 152 over 4 / 162 / 114 at 128 x 128; four groups of 2048 (N 1021, C 1019) 143 / 128 / 111
//   fp32 (N 2048, C 2048): one group of 4096 rows 679 / 413 / 377 / 366 / 289 (119 TFLOP/s), of 1024 172 / 106 / 99 / 109 / 160
// fp32 rows, whose products take their tile's time whether its rows are there or not, in tiles of 32 rows where the groups are shorter:
// 128 experts (N 1024, C 768, 403 MB) of 8 rows 210 / 178 / 146 / 136 / 212, 32 x 64 over 8 shares 134; of one row 204 / 177 / 147 / 137 / 212, 130;
// 16 experts of one row 29 / 25 / 26 / 33 / 61, 20.
template <typename T, Mode MODE, bool EIGHT = false>
static int any_t(const char* what, const ProductArgs& p, hipStream_t stream) {
    const int64_t tiles = even_tiles<MODE>(p, 64, 64), rows = even_rows(p);
    if (tiles <= 96) return any_go<T, MODE, EIGHT, 32, 32, 1, 1, 16>(what, p, stream);
    if constexpr (sizeof(T) == 4 && MODE != kWgrad)
        if (rows <= 32) return any_go<T, MODE, EIGHT, 32, 64, 1, 2, 8>(what, p, stream);
    if (tiles <= 256) return any_go<T, MODE, EIGHT, 64, 64, 2, 2, 4>(what, p, stream);
    if (tiles < 1024 || (MODE != kWgrad && rows <= 64)) return any_go<T, MODE, EIGHT, 64, 64, 2, 2, 2>(what, p, stream);
    return any_go<T, MODE, EIGHT, 128, 128, 2, 4, 1>(what, p, stream);
}

// ---------------------------------------------------------------- tiles through direct loads
typedef __amdgpu_buffer_rsrc_t Buffer;
typedef uint32_t u2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u4_t __attribute__((ext_vector_type(4)));
typedef int i4_t __attribute__((ext_vector_type(4)));
// An offset past every buffer's bytes: a load of it gives zeros, a store nothing
constexpr uint32_t kNone = 0x80000000u;
__device__ __forceinline__ Buffer buffer(const uint8_t* p) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p), 0, 0x7fffffff, 0x00020000);
}
// Direct load of 16 bytes per lane, from base + off + step, to lds + 16 lane (AUX 2: not kept in L2)
template <int AUX>
__device__ __forceinline__ void load16(Buffer base, uint32_t off, uint32_t step, uint8_t* __restrict lds) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(base, (lds_ptr_t)lds, 16, off, step, 0, AUX);
}

// An operand's stages: its pieces (16 bytes, 8 values) go straight into LDS, D loads of 64 pieces per wave and stage, RL stored rows each
template <typename T, int W, bool COL, int KB, int NW>
struct Loads {
    using S = Stage<T, W, COL, KB>;
    static constexpr int D = W * KB / 64 / NW, RL = 64 / S::PR;
    static_assert(W * KB % (64 * NW) == 0, "every wave the same loads");
    static __device__ __forceinline__ int row(int load) { return load * RL + (threadIdx.x & 63) / S::PR; }   // the lane's stored row in it
    static __device__ __forceinline__ int piece(int load) { return ((threadIdx.x & 63) % S::PR) ^ S::swizzle(row(load)); }
};

template <int BM, int BN, int NW, int ST, int KB, int OR>
struct TileShape {
    static constexpr int stage_b = (BM + BN) * KB * 16, out_b = OR * 128;   // (a wave's results, OR rows of 128 bytes at a time)
    static constexpr int smem = ST * stage_b + NW * out_b;
    static_assert(smem <= 160 * 1024, "LDS of a CU");
};

// A wave's LDS accesses before are done before those after, across its lanes (they complete in order)
__device__ __forceinline__ void wave_lds_order() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
    asm volatile("" ::: "memory");
}
// A uniform load through the scalar cache's counter, which the waits on vector loads do not count
__device__ __forceinline__ int uniform_load(const int32_t* p) { return *(const __attribute__((address_space(4))) int32_t*)p; }

struct TileGrid {
    int ny, per, nx;         // feature tiles, of a workgroup, row tiles (wgrad)
    int stream;              // weights that one row tile reads are not kept in L2
    int sorted;              // wgrad: the groups by size
    uint32_t nchunk;
    FastDiv blocks, divx;
};
constexpr int RB = 4;        // row tiles of a block

// BM rows x BN features per tile, `per` feature tiles of one row tile after one another in a workgroup of WM x WN waves. A stage is KB
// chunks (8 values) of the contracted values of every row, in a ring of ST slots that direct loads fill: offsets per lane from a base that moves
// with the stages, so that a load costs no address arithmetic, and an offset past the buffer where there is no such row, column or value: it
// reads nothing and leaves zeros, so that no operand is masked and the number of loads, which the waits count, is fixed. A wave multiplies FM x FN
// fragments of 32 x 32; the reads of the next step's operands and a part of the loads go between its products. The barrier at a stage's end
// comes before its last step, whose operands are in registers, and the next stage's first ones are read behind it. The stages of the feature
// tiles form one sequence: the next tile's first stages load while this one's results are written.
//
// What bounds it: with few rows to a group the weights' stream (20480 rows of 512 experts, N 1024, C 2048: 383 us, 5.7 TB/s over 2.1 GB of weights;
// 2030 rows, N 2560, C 640: 218 us, 7.4 TB/s); with many neither the loads nor the products alone, but how far they overlap: the loads alone bring in
// 23 bytes per clock and CU, whether the lines come from L2 or beyond (the L1 stands half of the time for lines under way), which would be 1.8
// PFLOP/s in tiles of 256 x 256 and 1.2 in 128 x 256; the products without the loads take 365 of the 476 to 493 us of one group of 8192 rows (N 8192,
// C 4096), 1115 to 1155 TFLOP/s. LDS is busy a quarter of the time, without conflicts. A group's last row tile costs a whole one: 8 experts (N, C
// 4096) of 2048 rows each 521 us, 1.05 PFLOP/s, of 1900 to 2196 575, matrix cores 57% busy; row gradients of 128 experts (N 2048, C 1024, fp16), 128
// x 256, of 512 rows each 347 us, of 513 400, of 576 410, of 640 430. The weights' gradients spill SGPRs (256 x 256 17, from 8-bit rows 14; 64 x 128
// 66 and 6), no VGPRs.
//
// Measured: four waves of 128 x 128 instead of eight 505 against 455 us (one group of 8192); stages of 64 values in two slots for the largest
// tile 476 against 450, of 32 values for 128 x 256 (half a line per row) 545 against 383 (20480 rows); 64 x 256 397, 128 x 128 430; row tiles of a
// group one by one instead of RB at a time 394 against 305 (loads alone); all groups' weights kept in L2 416 against 383. Without gain: another
// first stage in each workgroup, lines brought into L2 ahead (a load per line, 480 -> 610 us), other cache policies, longer rings.
template <typename T, Mode MODE, bool EIGHT, int BM, int BN, int WM, int WN, int ST, int KB, int OR, int OCC>
__global__ void __launch_bounds__(64 * WM * WN, OCC) k_product_tiles(ProductArgs p, TileGrid grid) {
    constexpr int NW = WM * WN, FM = BM / WM / 32, FN = BN / WN / 32, BK = KB * 8, SP = KB / 2;
    constexpr bool XCOL = MODE == kWgrad, YCOL = MODE != kProduct;
    using Sh = TileShape<BM, BN, NW, ST, KB, OR>;
    using LX = Loads<T, BM, XCOL, KB, NW>;
    using LY = Loads<T, BN, YCOL, KB, NW>;
    // (8-bit rows of a go through registers: CY pieces of 16 codes per thread and stage, NR rows of them per wave)
    constexpr int DX = LX::D, DY = EIGHT ? 0 : LY::D, D = DX + DY, CY = EIGHT ? BK * BN / (16 * 64 * NW) : 0, NR = 64 / (BN / 16);
    extern __shared__ __align__(16) uint8_t smem[];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    // Workgroup b runs on XCD b % 8 (the grid's rows are whole eights). Each XCD takes an eighth of the row tiles, neighbours, in blocks of RB with
    // their chunks of features: what runs at once on it reads few different rows of either operand. Where eighths would leave more than
    // a ninth of the chip idle, the blocks go over all XCDs.
    const uint32_t b = wide_block(), xcd = b & 7;
    int g, x0, xn, K, k_first = 0, chunk = 0;
    auto order = [&](uint32_t i, int tiles) INLINE {   // the row tile of workgroup i of those of that many row tiles (-1: none), and its chunk
        uint32_t block = grid.blocks(i), in = i - block * (RB * grid.nchunk), rows = RB;
        if (int(block) >= tiles / RB) {   // (the last block has fewer rows)
            in += (block - tiles / RB) * (RB * grid.nchunk);
            block = tiles / RB;
            rows = max(tiles % RB, 1);
        }
        chunk = int(in / rows);
        return chunk < int(grid.nchunk) && int(block * RB) < tiles ? int(block * RB + in % rows) : -1;
    };
    auto which = [&](int total) INLINE {
        const int each = (total + 7) / 8;
        if (each * 8 - total > total / 8) return order(b, total);
        const int first = int(xcd) * each, j = order(b >> 3, max(0, min(each, total - first)));
        return j < 0 ? -1 : first + j;
    };
    bool once = grid.stream;
    if constexpr (MODE == kWgrad) {
        int index;
        // The groups' sizes differ, and with them their tiles' work: the largest first, their row tiles round the XCDs (65536 rows of 128 experts
        // with 100 to 4800 each, 2048 x 1024: 389 us; in the groups' order 420, a group's tiles on one XCD 759). Short groups' time is their
        // results', which eighths write better (20480 rows of 512 experts, 1280 x 2560 fp32: 1255 against 1363).
        if (grid.sorted) {
            const int j = order(b >> 3, (p.E * grid.nx - int(xcd) + 7) / 8);
            index = j < 0 ? -1 : j * 8 + int(xcd);
        } else {
            index = which(p.E * grid.nx);
        }
        if (index < 0) return;
        const int rank = int(grid.divx(uint32_t(index)));
        g = grid.sorted ? group_by_size(p.bounds, p.E, p.M, rank) : rank;
        x0 = (index - rank * grid.nx) * BM;
        xn = min(BM, p.N - x0);
        k_first = p.bounds ? min(max(p.bounds[g], 0), p.M) : 0;
        K = max(0, (p.bounds ? min(max(p.bounds[g + 1], 0), p.M) : p.M) - k_first);
        if (K == 0 && p.add) return;
    } else {
        const RowTile t = find_tile<BM>(p.bounds, p.E, p.M, which);
        if (t.rows == 0) return;
        g = t.g;
        x0 = t.row0;
        xn = t.rows;
        K = MODE == kProduct ? p.C : p.N;
        once = once && t.only;
    }
    const int features = MODE == kProduct ? p.N : p.C, nst = EIGHT ? max(1, (K + 2 * BK - 1) / (2 * BK)) * 2 : max(1, (K + BK - 1) / BK);   // (8-bit rows: two by two)
    int ft = chunk * grid.per;
    const int ft1 = min(ft + grid.per, grid.ny);
    const bool gather = MODE == kWgrad && p.rows;

    // Where the lane's pieces come from: offsets from a base that moves from stage to stage. ROW operands: one per load, none where there is
    // no such row. COL ones: the lane's first row and column (none past the last column), a load's rows by a uniform step.
    const uint8_t *xb, *yb, *y0;
    uint32_t xo[XCOL ? 2 : DX], yo[YCOL ? 2 : DY];
    uint32_t xstep, ystep;   // from row to row, in bytes
    xstep = uint32_t(p.ldx * 2);
    ystep = uint32_t((MODE == kWgrad ? p.ldy : int64_t(p.C)) * 2);
    if constexpr (XCOL) {
        xb = static_cast<const uint8_t*>(p.x) + (int64_t(k_first) * p.ldx + x0) * 2;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int c = LX::piece(wave * DX + i) * 8;
            xo[i] = x0 + c < p.N ? lane / LX::S::PR * xstep + c * 2 : kNone;
        }
    } else {
        xb = static_cast<const uint8_t*>(p.x) + (p.rows ? 0 : x0 * p.ldx * 2);
#pragma unroll
        for (int i = 0; i < DX; ++i) {
            const int r = LX::row(wave * DX + i);
            uint32_t a = r;
            bool in = r < xn;
            if (p.rows) {
                a = uint32_t(p.rows[x0 + min(r, xn - 1)]);
                in = in && a < uint32_t(p.a_rows);
            }
            xo[i] = in ? a * xstep + LX::piece(wave * DX + i) * 16 : kNone;
        }
    }
    if constexpr (MODE == kWgrad)
        y0 = static_cast<const uint8_t*>(p.y) + (gather ? 0 : int64_t(k_first) * p.ldy * (EIGHT ? 1 : 2));
    else
        y0 = static_cast<const uint8_t*>(p.y) + int64_t(g) * p.N * p.C * 2;
    const uint8_t* const x0b = xb;
    int jf = ft, jst = 0, jslot = 0;   // the next stage to load: of feature tile jf, into slot jslot
    auto point = [&]() INLINE {
        xb = x0b;
        if constexpr (EIGHT) return;
        if constexpr (YCOL) {
            yb = y0 + int64_t(jf) * BN * 2;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int c = LY::piece(wave * DY + i) * 8;
                yo[i] = jf * BN + c < p.C ? (gather ? 0 : lane / LY::S::PR * ystep) + c * 2 : kNone;
            }
        } else {
            yb = y0 + int64_t(jf) * BN * p.C * 2;
#pragma unroll
            for (int i = 0; i < DY; ++i) {
                const int r = LY::row(wave * DY + i);
                yo[i] = jf * BN + r < p.N ? r * ystep + LY::piece(wave * DY + i) * 16 : kNone;
            }
        }
    };
    point();
    // gather: the rows of a's rows of the next stage, a stage ahead
    constexpr int NI = MODE == kWgrad && !EIGHT ? DY * LY::RL : 1;
    int index[NI] = {};
    auto fetch = [&]() INLINE {
        if (MODE == kWgrad && !EIGHT && gather && K > 0) {
            const int k = k_first + jst * BK + wave * NI;
#pragma unroll
            for (int i = 0; i < NI; ++i) index[i] = uniform_load(p.rows + min(k + i, p.M - 1));
        }
    };
    fetch();
    // 8-bit rows of a go through registers, since they have to become values of T, as many bytes again, on the way: a stage's codes are loaded two
    // stages ahead into one of two sets (loads complete in order, so a wait for newer codes would wait for the operands behind them, too), the
    // rows' indices two stages before those, and written between the products that follow the barrier that frees their slot (zeros past
    // the group's rows and a's columns, and for a row that there is not). 65536 rows of 128 experts, 2048 x 1024: 425 us against 403 from rows in
    // 16 bits; with one set 515, with indices in scalar registers, whose loads share a counter with LDS, 525; through the 64 x 64 tiles 1292.
    const uint32_t blocks = uint32_t(p.C) / 32;
    const uint8_t* const s0 = EIGHT ? p.scales + (gather ? 0 : int64_t(k_first) * blocks) : nullptr;
    int ef = ft, est = 0;   // the feature tile and stage whose codes are loaded next
    i4_t codes[2][EIGHT ? CY : 1];
    uint32_t scales[2][EIGHT ? CY : 1], picks[2][EIGHT ? CY : 1];
    auto pick8 = [&](int set, int st) INLINE {   // stage st's rows of a (in every call, so that the waits can count on it)
        uint32_t ln = lane;
        asm volatile("" : "+v"(ln));   // (addresses formed here, not all kept)
        const Buffer rb = buffer(reinterpret_cast<const uint8_t*>(p.rows + (gather ? int64_t(k_first) + int64_t(st) * BK : 0)));
        const int lim = gather ? K - st * BK : 0;
#pragma unroll
        for (int i = 0; i < CY; ++i) {
            const int k = (i * NW + wave) * NR + ln / (BN / 16);
            picks[set][i] = __builtin_amdgcn_raw_buffer_load_b32(rb, k < lim ? uint32_t(k) * 4 : kNone, 0, 0);
        }
    };
    auto fetch8 = [&](int set) INLINE {
        uint32_t ln = lane;
        asm volatile("" : "+v"(ln));
        const int k0 = est * BK, lim = ef < ft1 ? K - k0 : 0;
        const Buffer qb = buffer(y0 + (gather ? 0 : int64_t(k0) * p.C)), sb = buffer(s0 + (gather ? 0 : int64_t(k0) * blocks));
#pragma unroll
        for (int i = 0; i < CY; ++i) {
            const int k = (i * NW + wave) * NR + ln / (BN / 16), c = ef * BN + ln % (BN / 16) * 16;
            const uint32_t a = gather ? picks[set][i] : uint32_t(k);
            const bool in = (k < lim) & (c < p.C) & (!gather | (a < uint32_t(p.a_rows)));
            uint32_t qo = in ? a * uint32_t(p.C) + c : kNone, so = in ? a * blocks + c / 32 : kNone;
            asm volatile("" : "+v"(qo), "+v"(so));   // (one load whatever `in` is: with one on each side of a branch the second waits for the first)
            codes[set][i] = __builtin_bit_cast(i4_t, __builtin_amdgcn_raw_buffer_load_b128(qb, qo, 0, 0));
            scales[set][i] = __builtin_amdgcn_raw_buffer_load_b8(sb, so, 0, 0);
        }
        pick8(set, est + 2 < nst ? est + 2 : est + 2 - nst);
        if (++est == nst) {
            est = 0;
            ++ef;
        }
    };
    auto put8 = [&](int set, int half) INLINE {   // eight codes (one of 2 CY)
        uint32_t ln = lane;
        asm volatile("" : "+v"(ln));
        const int i = half / 2, h = half % 2, k = (i * NW + wave) * NR + ln / (BN / 16), c = ln % (BN / 16) * 2;
        const auto f = mx8_values(codes[set][i][2 * h], codes[set][i][2 * h + 1], mx8_scale(scales[set][i]));
        *reinterpret_cast<Vec<T>*>(smem + jslot * Sh::stage_b + BM * KB * 16 + LY::S::piece(k, c + h)) = __builtin_convertvector(f, Vec<T>);
    };
    if constexpr (EIGHT) {
        pick8(0, 0);
        pick8(1, 1);
        fetch8(0);
        fetch8(1);
    }
    // Load i of the next stage; past the last stage of the last feature tile zeros are loaded that nothing reads, so that the waits
    // can count on every load.
    auto load_y = [&](uint32_t off, uint32_t step, uint8_t* l) INLINE {
        if (MODE != kWgrad && once)
            load16<2>(buffer(yb), off, step, l);
        else
            load16<0>(buffer(yb), off, step, l);
    };
    auto load = [&](int i) INLINE {
        uint32_t xs = xstep, ys = ystep;
        asm volatile("" : "+s"(xs), "+s"(ys));   // (steps formed here, not all kept in registers)
        uint8_t* const s = smem + jslot * Sh::stage_b;
        const int lim = jf < ft1 ? K - jst * BK : 0;   // the stage's values (rows) before the end
        if (i < DX) {
            const int at = wave * DX + i;
            if constexpr (XCOL)
                load16<0>(buffer(xb), LX::row(at) < lim ? xo[i & 1] : kNone, uint32_t(at * LX::RL) * xs, s + at * 1024);
            else
                load16<0>(buffer(xb), LX::piece(at) * 8 < lim ? xo[i % DX] : kNone, 0, s + at * 1024);
        } else {
            const int j = i - DX, at = wave * DY + j;
            uint8_t* const l = s + BM * KB * 16 + at * 1024;
            if constexpr (MODE == kProduct) {
                load_y(LY::piece(at) * 8 < lim ? yo[j % DY] : kNone, 0, l);
            } else if (gather) {
                int a = -1;
#pragma unroll
                for (int r = 0; r < LY::RL; ++r) a = lane / LY::S::PR == r ? index[(j * LY::RL + r) % NI] : a;
                const bool in = LY::row(at) < lim && uint32_t(a) < uint32_t(p.a_rows) && yo[j & 1] != kNone;
                load_y(in ? uint32_t(a) * ys + yo[j & 1] : kNone, 0, l);
            } else {
                load_y(LY::row(at) < lim ? yo[j & 1] : kNone, uint32_t(at * LY::RL) * ys, l);
            }
        }
    };
    auto advance = [&]() INLINE {   // all loads of the stage are issued: on to the next one
        jslot = jslot == ST - 1 ? 0 : jslot + 1;
        ++jst;
        xb += XCOL ? int64_t(BK) * p.ldx * 2 : BK * 2;
        if (!gather && !EIGHT) yb += YCOL ? int64_t(BK) * (MODE == kWgrad ? p.ldy : int64_t(p.C)) * 2 : BK * 2;
        if (jst == nst) {
            jst = 0;
            ++jf;
            point();
        }
        fetch();
    };

    const int wm = wave / WN * FM * 32, wn = wave % WN * FN * 32;
    struct Ops {
        Vec<T> b[FN], a[FM];
    };
    f16_t acc[FM][FN];
    auto read = [&](Ops& o, int slot, int t, int i) INLINE {   // operand i of step t
        const uint8_t* const s = smem + slot * Sh::stage_b;
        if (i < FN)
            o.b[i % FN] = LY::S::read(s + BM * KB * 16, wn + 32 * i, t);
        else
            o.a[(i - FN) % FM] = LX::S::read(s, wm + 32 * (i - FN), t);
    };
    // A step's products, row by row, with the reads of the next step's operands and part `part` (of SP) of the next stage's loads between them
    auto step = [&](auto on, const Ops& o, Ops& next, int slot, int t, int part, int set) INLINE {
#pragma unroll
        for (int m = 0; m < FM; ++m) {
            if constexpr (decltype(on)::value) {
#pragma unroll
                for (int f = 0; f < FN; ++f) acc[m][f] = mma(o.b[f], o.a[m], acc[m][f]);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < FM + FN; ++i)
                    if (i >= m * (FM + FN) / FM && i < (m + 1) * (FM + FN) / FM) read(next, slot, t, i);
            }
#pragma unroll
            for (int i = 0; i < D; ++i)
                if (i >= (part * FM + m) * D / (SP * FM) && i < (part * FM + m + 1) * D / (SP * FM)) load(i);
            if constexpr (EIGHT)
                if (part == 0) {
#pragma unroll
                    for (int h = 0; h < 2 * CY; ++h)
                        if (h >= m * 2 * CY / FM && h < (m + 1) * 2 * CY / FM) put8(set, h);
                    if (m == FM - 1) fetch8(set);
                }
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    // Waits count the loads: at the end of a stage those of ST - 2 stages were issued behind the next one's, and in a feature tile's first ST
    // - 2 stages the stores of the tile before, where these are of whole pieces (at least kStores per wave whatever is inside; none are counted on
    // with add, nor of a feature tile that ends inside a piece, whose single values may be fewer).
    constexpr int kStage = D + 3 * CY, kStores = FM * FN * 2, kCap = 63;
    auto landed = [&](bool stores) INLINE {
        if (stores)
            wait_vm<(kStage * (ST - 2) + kStores < kCap ? kStage * (ST - 2) + kStores : kCap)>();
        else
            wait_vm<(kStage * (ST - 2) < kCap ? kStage * (ST - 2) : kCap)>();
    };
    bool stored = false;   // the tile before left kStores stores or more under way
    auto finish = [&]() INLINE {
        // The results through LDS, OR rows of QP fourths of a fragment (8 features each) at a time, so that whole lines are stored. Lane l's
        // value i of a fragment: feature 8 (i / 4) + 4 (l / 32) + i % 4, row l % 32.
        auto results = [&](auto staged, auto zero, auto added) INLINE {
            constexpr bool ADD = decltype(added)::value;   // (in fp32 up to the sum, of the result's type then)
            typedef decltype(staged) O;
            typedef decltype(zero) R;
            constexpr int sz = sizeof(O), QP = 16 / sz < 4 * FN ? 16 / sz : 4 * FN, V = 16 / sz;
            constexpr int PR = QP * 8 / V, NP = OR * PR / 64;   // pieces of 16 bytes in a row, of a lane; in LDS piece p of row r is at p ^ (r / 2 % 8)
            static_assert(4 * FN % QP == 0 && FM * (4 * FN / QP) * NP * (32 / OR) >= kStores, "the stores of a wave");
            typedef O vec4 __attribute__((ext_vector_type(4)));
            uint8_t* const w = smem + ST * Sh::stage_b + wave * Sh::out_b;
            R* const out = static_cast<R*>(p.out) + (MODE == kWgrad ? int64_t(g) * p.N * p.C : 0) + x0 * p.ldout;
            const bool whole = features % V == 0 || (ft + 1) * BN <= features;   // the feature tile ends with a piece
            stored = !ADD && whole;
            const Buffer to_out = __builtin_amdgcn_make_buffer_rsrc(out, 0, int(((xn - 1) * p.ldout + features) * sizeof(R)), 0x00020000);
#pragma unroll
            for (int m = 0; m < FM; ++m) {
#pragma unroll
                for (int q = 0; q < 4 * FN; q += QP) {
#pragma unroll
                    for (int e = q / 4; e <= (q + QP - 1) / 4; ++e) asm volatile("" : "+a"(acc[m][e]));   // (read one piece at a time)
#pragma unroll
                    for (int pass = 0; pass < 32 / OR; ++pass) {
                        int ln = lane;
                        asm volatile("" : "+v"(ln));   // (addresses formed piece by piece, not all kept from before the loop)
#pragma unroll
                        for (int i = 0; i < QP; ++i) {
                            if (OR < 32 && (ln & 31) / OR != pass) break;
                            vec4 v;
#pragma unroll
                            for (int e = 0; e < 4; ++e) v[e] = O(acc[m][(q + i) / 4][(q + i) % 4 * 4 + e]);
                            const int b = (8 * i + 4 * (ln >> 5)) * sz, r = ln % OR;
                            *reinterpret_cast<vec4*>(w + r * 128 + (((b >> 4) ^ (r / 2 % 8)) << 4) + (b & 15)) = v;
                        }
                        wave_lds_order();
                        asm volatile("" : "+v"(ln));
                        const int c = ft * BN + wn + q * 8 + ln % PR * V;
                        const int r0 = wm + 32 * m + pass * OR + ln / PR;
                        auto from = [&](int i) INLINE {
                            const int r = ln / PR + i * (64 / PR);
                            return w + r * 128 + ((ln % PR ^ (r / 2 % 8)) << 4);
                        };
                        if constexpr (ADD) {
                            // Four results a lane, whole ones (C is a multiple of eight); what is there is read for NP rows before the first
                            // is written. 20480 rows of 512 experts, 1280 x 2560: fp32 2.59 ms (13.4 GB read and written; row by row
                            // 3.48), bf16 2.44 (2.66), which waits for the stores of the step before; with steps read ahead 2.58 and 2.18, but registers spill
                            typedef R vec __attribute__((ext_vector_type(4)));
                            typedef std::conditional_t<sizeof(R) == 4, u4_t, u2_t> Raw;
                            uint32_t to[NP];
                            Raw old[NP];
#pragma unroll
                            for (int i = 0; i < NP; ++i) {
                                const int r = r0 + i * (64 / PR);
                                to[i] = r < xn && c < features ? uint32_t(r * int(p.ldout) + c) * sizeof(R) : kNone;
                                asm volatile("" : "+v"(to[i]));
                                if constexpr (sizeof(R) == 4)
                                    old[i] = __builtin_amdgcn_raw_buffer_load_b128(to_out, to[i], 0, 2);
                                else
                                    old[i] = __builtin_amdgcn_raw_buffer_load_b64(to_out, to[i], 0, 2);
                            }
                            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                            for (int i = 0; i < NP; ++i) {
                                const f4_t v = *reinterpret_cast<const f4_t*>(from(i)) + __builtin_convertvector(__builtin_bit_cast(vec, old[i]), f4_t);
                                const Raw raw = __builtin_bit_cast(Raw, __builtin_convertvector(v, vec));
                                if constexpr (sizeof(R) == 4)
                                    __builtin_amdgcn_raw_buffer_store_b128(raw, to_out, to[i], 0, 2);
                                else
                                    __builtin_amdgcn_raw_buffer_store_b64(raw, to_out, to[i], 0, 2);
                            }
                        } else if (whole) {
                            i4_t v[NP];
#pragma unroll
                            for (int i = 0; i < NP; ++i) v[i] = *reinterpret_cast<const i4_t*>(from(i));
#pragma unroll
                            for (int i = 0; i < NP; ++i) {
                                const int r = r0 + i * (64 / PR);
                                const uint32_t to = r < xn && c < features ? uint32_t(r * int(p.ldout) + c) * sz : kNone;
                                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4_t, v[i]), to_out, to, 0, 2);   // (non-temporal)
                            }
                        } else {   // the last feature tile, cut short inside a piece
                            for (int i = 0; i < NP && r0 + i * (64 / PR) < xn; ++i)
                                for (int e = 0; e < V && c + e < features; ++e)
                                    out[(r0 + i * (64 / PR)) * p.ldout + c + e] = *reinterpret_cast<const O*>(from(i) + e * sz);
                        }
                        wave_lds_order();
                    }
                }
            }
        };
        auto as = [&](auto zero) INLINE {
            if (MODE == kWgrad && p.add)
                results(float(), zero, std::true_type());
            else
                results(zero, zero, std::false_type());
        };
        if (p.out_type == FRT_GGML_F32)
            as(float());
        else if (p.out_type == FRT_GGML_F16)
            as(_Float16());
        else
            as(__bf16());
    };
#pragma unroll(EIGHT ? ST - 1 : 1)
    for (int s = 0; s < ST - 1; ++s) {
#pragma unroll
        for (int i = 0; i < D; ++i) load(i);
        if constexpr (EIGHT) {
#pragma unroll
            for (int h = 0; h < 2 * CY; ++h) put8(s & 1, h);
            fetch8(s & 1);
        }
        advance();
    }
#pragma unroll
    for (int i = 0; i < D / SP; ++i) load(i);
    if constexpr (EIGHT) {
#pragma unroll
        for (int h = 0; h < 2 * CY; ++h) put8((ST - 1) & 1, h);
        fetch8((ST - 1) & 1);
    }
    wait_vm<(kStage * (ST - 2) + D / SP < kCap ? kStage * (ST - 2) + D / SP : kCap)>();
    ring_barrier();
    int slot = 0;
    Ops o[2];
#pragma unroll
    for (int i = 0; i < FM + FN; ++i) read(o[0], 0, 0, i);
    lds_reads_done();   // (nothing pending where the loop is entered: its waits are then for its own reads)
    for (; ft < ft1; ++ft) {
        // (a wave that has no rows or features in the tile only loads)
        const bool live = wm < xn && ft * BN + wn < features;
#pragma unroll
        for (int m = 0; m < FM; ++m)
#pragma unroll
            for (int f = 0; f < FN; ++f)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[m][f][i] = 0.0f;
        auto stage = [&](auto on, int st, int set) INLINE {
#pragma unroll
            for (int t = 0; t < SP - 1; ++t) step(on, o[t & 1], o[(t & 1) ^ 1], slot, t + 1, t + 1, set);
            advance();
            // the end of the stage: the next one has landed, all waves have read this one, and its slot is loaded anew
            landed(st < ST - 2 && stored);
            ring_barrier();
            slot = slot == ST - 1 ? 0 : slot + 1;
            step(on, o[(SP - 1) & 1], o[0], slot, 0, 0, set);   // (past the last stage it reads what nothing uses)
        };
        auto stages = [&](auto on) INLINE {
            if constexpr (EIGHT) {
                for (int st = 0; st < nst; st += 2) {   // (two by two, so that the registers of each set are known)
                    stage(on, st, ST & 1);
                    stage(on, st + 1, (ST & 1) ^ 1);
                }
            } else {
                for (int st = 0; st < nst; ++st) stage(on, st, 0);
            }
        };
        if (live)
            stages(std::true_type());
        else
            stages(std::false_type());
        stored = false;
        if (live) finish();
    }
    // no load into LDS is under way when the workgroup ends (the last tile's stores may be)
    if (stored)
        wait_vm<(kStores < kCap ? kStores : kCap)>();
    else
        wait_vm<0>();
}

template <typename T, Mode MODE, bool EIGHT, int BM, int BN, int WM, int WN, int ST, int KB, int OR, int OCC>
static int tiles_go(const char* what, const ProductArgs& p, hipStream_t stream) {
    const int features = MODE == kProduct ? p.N : p.C, ny = (features + BN - 1) / BN, nx = (p.N + BM - 1) / BM;
    const bool grouped = p.bounds != nullptr;
    const int64_t groups = grouped ? std::min(p.E, std::max(p.M, 1)) : 1;
    const bool sorted = MODE == kWgrad && grouped && p.E <= 512 && p.M / groups >= 128;
    // feature tiles of a workgroup: about kStages stages, as long as kFill workgroups remain (half a tile of each group empty)
    const int64_t tiles = MODE == kWgrad ? int64_t(p.E) * nx : tiles_at_most(p.M, p.E, BM, grouped);
    const int64_t likely = MODE == kWgrad ? tiles : grouped ? std::max<int64_t>(p.M / BM + groups / 2, groups) : tiles;
    const int64_t K = MODE == kProduct ? p.C : MODE == kGrad ? p.N : p.M / groups;
    const int nst = int(std::max<int64_t>(1, (K + KB * 8 - 1) / (KB * 8)));
    // (in units of 64 values: a workgroup takes about 4 us to begin and end. 40 / 64 / 128 and at least 512 workgroups: 20480 rows, C 2048, 382 / 381 /
    // 381 us; 2030 rows, C 640, 218 / 218 / 248; 640 rows, C 2048, 227 / 235 / 255; rows' gradients of 17770, N 2048, 187 / 209 / 209. Weights'
    // gradients of groups by size, 65536 rows: 8 / 16 / 32 425 / 389 / 569; short ones 1259 / 1300 / 1296)
    constexpr int kFill = 512;
    const int kStages = (MODE == kWgrad ? sorted ? 16 : 8 : 40) * 8 / KB;
    int nchunk = std::max(1, std::min(kStages / nst, ny));
    nchunk = (ny + nchunk - 1) / nchunk;
    while (nchunk < ny && likely * nchunk < kFill) ++nchunk;
    const int per = (ny + nchunk - 1) / nchunk;
    nchunk = (ny + per - 1) / per;
    const int64_t wgs = (tiles + 7) / 8 * 8 * nchunk;
    if (wgs > 0x7ffff000 || tiles > 0x7ffff000) return set_error(kErrShape, "%s: M=%d N=%d C=%d E=%d", what, p.M, p.N, p.C, p.E);
    const uint32_t y = uint32_t((wgs + (1 << 22) - 1) >> 22), x = uint32_t(((wgs + y - 1) / y + 7) / 8 * 8);   // (fewer than 2^32 threads in a dimension)
    constexpr int smem = TileShape<BM, BN, WM * WN, ST, KB, OR>::smem;
    FRT_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(&k_product_tiles<T, MODE, EIGHT, BM, BN, WM, WN, ST, KB, OR, OCC>),
                                hipFuncAttributeMaxDynamicSharedMemorySize, smem));
    const TileGrid grid{ny, per, nx, MODE != kWgrad, sorted, uint32_t(nchunk), FastDiv(uint32_t(RB * nchunk)), FastDiv(uint32_t(nx))};
    launch_timed(what, k_product_tiles<T, MODE, EIGHT, BM, BN, WM, WN, ST, KB, OR, OCC>, dim3(x, y), dim3(64 * WM * WN), smem, stream, p, grid);
    FRT_LAUNCHED(what);
    return kOk;
}

// ---------------------------------------------------------------- few rows
__device__ __forceinline__ f4_t mma16(Vec<_Float16> w, Vec<_Float16> x, f4_t acc) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(w, x, acc, 0, 0, 0); }
__device__ __forceinline__ f4_t mma16(Vec<__bf16> w, Vec<__bf16> x, f4_t acc) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, x, acc, 0, 0, 0); }

// 16 features x 16 rows by KW waves that share the values of a row, straight from global memory into the registers of the matrix
// instructions. The weights are the first operand, so that a lane's four results are adjacent features of one row. A group of 128 values is 16
// chunks: step i multiplies chunks 4 i + l / 16 of lane l's feature and row. Wave w takes the groups w, w + KW, ..., two at a time in
// flight; the waves' sums are added in their order. Rows and features past the end are the last one again, never stored. Bound by the chain of
// trips to memory (bounds, then the row's index and the weights, then the activations): one token's ten experts (N 1024, C 2048, 42 MB)
// 12.3 us; weights not kept in L2 13.3.
template <typename T, int KW>
__global__ void __launch_bounds__(256) k_product_rows(ProductArgs p, int ntile, FastDiv ntiles) {
    constexpr int FW = 4 / KW, V = Chunk<T>::V, P = 2;   // tiles of a workgroup; groups in flight (four: 5% slower)
    __shared__ f4_t s_sum[4][64];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, j = lane & 15, g = lane >> 4;
    const int kw = wave % KW;
    const uint32_t unit = wide_block() * FW + wave / KW, tile = ntiles(unit);
    const RowTile t = find_tile<16>(p.bounds, p.E, p.M, [&](int total) { return int(tile) < total ? int(tile) : -1; });
    const int f0 = int(unit - tile * ntile) * 16, nc = p.C / V, ng = (nc + 15) / 16;
    f4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
    if (t.rows > 0) {   // (uniform over the wave)
        const int r = t.row0 + min(j, t.rows - 1);
        int a = r;
        if (p.rows) a = gld<int>(p.rows + r);   // (under way while the weights' loads are issued)
        const T* const w = static_cast<const T*>(p.y) + (int64_t(t.g) * p.N + min(f0 + j, p.N - 1)) * p.C;
        struct Group {
            Vec<T> w[4], x[4];
        } u[P];
        auto load_w = [&](int q, Group& o) INLINE {   // (chunks past the last are the last again: its partner is zeros there)
#pragma unroll
            for (int i = 0; i < 4; ++i) o.w[i] = gld<Vec<T>>(w + min(16 * q + 4 * i + g, nc - 1) * V);
        };
        const T* x = nullptr;
        auto load_x = [&](int q, Group& o) INLINE {
#pragma unroll
            for (int i = 0; i < 4; ++i) o.x[i] = gld<Vec<T>>(x + min(16 * q + 4 * i + g, nc - 1) * V);
        };
        bool ok = false;   // the lane's row is one of a's (else zeros, as a factor: an infinite weight gives NaN in every kernel)
        auto multiply = [&](int q, const Group& o) INLINE {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool in = 16 * q + 4 * i + g < nc;
                const Vec<T> zero = {};
                acc = mma16(in ? o.w[i] : zero, in && ok ? o.x[i] : zero, acc);
            }
        };
#pragma unroll
        for (int k = 0; k < P; ++k)
            if (kw + k * KW < ng) load_w(kw + k * KW, u[k]);
        __builtin_amdgcn_sched_barrier(0);
        ok = unsigned(a) < unsigned(p.a_rows);
        x = static_cast<const T*>(p.x) + int64_t(ok ? a : 0) * p.ldx;
#pragma unroll
        for (int k = 0; k < P; ++k)
            if (kw + k * KW < ng) load_x(kw + k * KW, u[k]);
        for (int q = kw; q < ng; q += P * KW) {
#pragma unroll
            for (int k = 0; k < P; ++k) {
                const int c = q + k * KW, n = c + P * KW;
                if (c < ng) multiply(c, u[k]);
                if (n < ng) {
                    load_w(n, u[k]);
                    load_x(n, u[k]);
                }
            }
        }
    }
    if constexpr (KW > 1) {
        s_sum[wave][lane] = acc;
        __syncthreads();
        if (kw != 0) return;
#pragma unroll
        for (int i = 1; i < KW; ++i) acc += s_sum[wave + i][lane];
    }
    if (j < t.rows && f0 + 4 * g < p.N) store4(p, (int64_t(t.row0) + j) * p.ldout + f0 + 4 * g, acc, p.N - f0 - 4 * g);
}

template <typename T, int KW>
static int rows_go(const ProductArgs& p, hipStream_t stream) {
    const int ntile = (p.N + 15) / 16;
    const int64_t units = tiles_at_most(p.M, p.E, 16, p.bounds != nullptr) * ntile, wgs = (units + 4 / KW - 1) / (4 / KW);
    if (units > 0x7ffff000) return set_error(kErrShape, "moe_product: M=%d N=%d E=%d", p.M, p.N, p.E);
    launch_timed("moe_product", k_product_rows<T, KW>, wide_grid(uint32_t(wgs)), dim3(256), 0, stream, p, ntile, FastDiv(uint32_t(ntile)));
    FRT_LAUNCHED("moe_product");
    return kOk;
}

// Whether the tiles through direct loads take a call: operands in whole, aligned pieces, offsets within 31 bits
template <typename T>
static bool pieces(const ProductArgs& p, int x_cols, bool wgrad) {
    const auto whole = [](const void* q, int64_t ld) { return reinterpret_cast<uintptr_t>(q) % 16 == 0 && ld % 8 == 0; };
    const auto near = [](int64_t rows, int64_t ld) { return ld < (int64_t(1) << 30) / std::max<int64_t>(rows, 1); };   // (twice as many bytes)
    return sizeof(T) == 2 && x_cols % 8 == 0 && p.C % 8 == 0 && whole(p.x, p.ldx) && whole(p.y, p.ldy) && near(512, p.ldout) &&
           near(wgrad || !p.rows ? 256 : p.a_rows, p.ldx) && near(wgrad && p.rows ? p.a_rows : 256, p.ldy);
}
template <typename T, Mode MODE, bool EIGHT = false>
static int tiles_t(const char* what, const ProductArgs& p, hipStream_t stream) {
    const int64_t rows = even_rows(p);
    const auto tiles = [&](int64_t BM, int64_t BN) { return even_tiles<MODE>(p, BM, BN); };
    // As few tiles as leave CUs idle share the summed values out. us, so / in tiles of 64 x 128: row gradients, one row (N 1024, C 2048) 8.2 / 12.1,
    // 16 rows (N 2560, C 640) 11.7 / 22.6, 2048 rows (512 x 512) 8.4 / 9.4; weights' gradients, one group of 8192 rows (512 x 512) 33 / 83,
    // of 2048 10.7 / 26.3. Just beyond: 16 groups of a row (N 768, C 2048) 13.0 / 12.1, 8 groups of 2048 rows 28.9 / 27.5
    if (tiles(64, 64) <= 256) return any_t<T, MODE, EIGHT>(what, p, stream);
    // us at 256 x 256 / 128 x 256 / 64 x 128:
    //   16384 rows of 8 experts (N, C 4096) 570 / 592; 65536 of 128 (N 2048, C 1024) 363 / 370 / 479; one group of 8192 (N 8192, C 4096) 488 / 521
    //   20480 rows of 512 experts (N 1024, C 2048) 555 / 383 / 416; 2030 rows (N 2560, C 640) 358 / 230 / 221; 640 rows 345 / 247 / 228
    //   one group of 2048 rows (N, C 2560) 61 / 36 / 48, of 512 61 / 36 / 22; 8 experts of 64 rows (N, C 2048) 48 / 31 / 22
    //   weights' gradients: 65536 rows of 128 experts 389 / 475; 8192 of 128 (1024 x 1024) 139 / 138 / 143; one group of 4096 (768 x 1408) 94 / 58 / 41
    if constexpr (MODE == kWgrad) {
        if (tiles(256, 256) >= 256)
            return tiles_go<T, MODE, EIGHT, 256, 256, 2, 4, 4, 4, 32, 2>(what, p, stream);
    } else {
        if (rows >= 1024 && tiles(256, 256) >= 512) return tiles_go<T, MODE, EIGHT, 256, 256, 2, 4, 4, 4, 32, 2>(what, p, stream);
        if (rows > 16 && tiles(128, 256) >= 128) return tiles_go<T, MODE, EIGHT, 128, 256, 2, 4, 3, 8, 16, 2>(what, p, stream);
    }
    return tiles_go<T, MODE, EIGHT, 64, 128, 2, 2, 3, 8, 16, 2>(what, p, stream);
}

template <typename T>
static int product_t(const ProductArgs& p, hipStream_t stream) {
    if constexpr (sizeof(T) == 2)
        if (pieces<T>(p, p.C, false)) {
            // The weights that tiles of 16 rows read: up to 256 MB straight into registers, beyond in tiles through LDS; a row's values over four
            // waves, or two, while the call has no more than three waves to a SIMD with that and each of them a group of values. us, four / two / one
            // wave to a row / tiles, weights from memory: experts of a row, N 1024, C 2048, 10 of them (640 units) 14.6 / 15.6 / 18.5 / 20.9, 12 15.1
            // / 16.0 / 19.1 / 21.5, 16 20.3 / 18.9 / 21.1 / 24.5, 24 27.4 / 23.9 / 26.3 / 23.6, 32 36 / 32 / 32 / 27, 64 (268 MB) 63 / 70 / 63 / 53;
            // C 512, 16 of them 8.6 / 7.1 / 6.9 / 11.7, 32 15.9 / 14.4 / 11.7 / 13.2; N 2560, C 640, 8 of them (1280 units) 11.6 / 10.5 / 11.4 /
            // 12.0, 9 12.9 / 10.9 / 11.4, 10 14.7 / 13.9 / 12.3 / 12.3, 32 37 / 29 / 27 / 29; N 2048, C 4096, 6 (768) 22 / 26 / 30 / 29, 12 (1536) 43
            // / 45 / 48 / 46, 13 48 / 53 / 50 / 47; one group of a row, C 4096, N 8192 17.8 / 19.3 / 30.6 / 28.7, N 16384 29.5 / 34.0 / 39.5 / 36.8.
            // Weights that more than one tile reads, up to 32 MB. us, so / in tiles: one group of 256 rows (N 512, C 1024, 17 MB) 7.4 /
            // 8.2, of 128 (N 1024, C 2048, 34 MB) 9.7 / 10.0, of 2048 (512 x 512, 67 MB) 17.2 / 8.3, of 256 (N 2048, C 2048, 134 MB) 31 / 15
            constexpr int kFew = 3 * 4 * 256;   // waves
            const int64_t rows = even_rows(p), units = even_tiles<kProduct>(p, 16, 16);
            if (units <= (int64_t(rows <= 16 ? 256 : 32) << 20) / 32 / p.C)
                return 4 * units <= kFew && p.C >= 512 ? rows_go<T, 4>(p, stream) : 2 * units <= kFew && p.C >= 256 ? rows_go<T, 2>(p, stream) : rows_go<T, 1>(p, stream);
            return tiles_t<T, kProduct>("moe_product", p, stream);
        }
    return any_t<T, kProduct>("moe_product", p, stream);
}
template <typename T>
static int grad_t(const ProductArgs& p, hipStream_t stream) {
    if constexpr (sizeof(T) == 2)
        if (pieces<T>(p, p.N, false)) return tiles_t<T, kGrad>("moe_product_grad", p, stream);
    return any_t<T, kGrad>("moe_product_grad", p, stream);
}
template <typename T>
static int wgrad_t(const ProductArgs& p, hipStream_t stream) {
    if constexpr (sizeof(T) == 2)
        if (pieces<T>(p, p.N, true))
            return p.scales ? tiles_t<T, kWgrad, true>("moe_product_wgrad", p, stream) : tiles_t<T, kWgrad>("moe_product_wgrad", p, stream);
    return p.scales ? any_t<T, kWgrad, true>("moe_product_wgrad", p, stream) : any_t<T, kWgrad>("moe_product_wgrad", p, stream);
}

int moe_product(int type, const ProductArgs& p, hipStream_t stream) { return FRT_BY_TYPE(type, product_t, p, stream); }
int moe_product_grad(int type, const ProductArgs& p, hipStream_t stream) { return FRT_BY_TYPE(type, grad_t, p, stream); }
int moe_product_wgrad(int type, const ProductArgs& p, hipStream_t stream) { return FRT_BY_TYPE(type, wgrad_t, p, stream); }

}  // namespace frt
