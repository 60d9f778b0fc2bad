// Products of the sorted rows with their experts' matrices, and both gradients, on the matrix cores: operands of 32 or 16 bits, sums in fp32.
//
//   product   out[r] = w_g a(r)          contracted over C, both operands' rows
//   grad      da[r] = w_g^T dout[r]      contracted over N: w's columns
//   wgrad     dw_g = sum_r dout[r] a(r)^T   contracted over the group's rows: columns of both
// r in [bounds[g], bounds[g + 1]); a(r) is row r, or row rows[r]. In all three an output tile is X Y^T with X the operand along the output's
// rows and Y the one along its columns ("features").
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

// A stage of an operand in LDS: W rows (or columns) of 128 bytes of contracted values, eight chunks of which step t takes 2 t and 2 t + 1 (one
// per lane half). ROW: [W][128 bytes], chunk c of row r at c ^ (r / 2 % 8), so that the sixteen rows of a read phase take sixteen different
// columns of the banks. COL: [128 / sizeof(T)][W], the contracted values apart: chunks of 16 bits are read by the transposing LDS read, four
// values of sixteen columns at a time (a lane's address is a quarter of one row's 32 bytes), 32-bit ones value by value; 32-byte
// blocks of rows that a read takes together lie in different banks.
template <typename T, int W, bool COL>
struct Stage {
    static constexpr int V = Chunk<T>::V, BK = 128 / int(sizeof(T)), bytes = W * 128;
    static constexpr int row_b = COL ? W * int(sizeof(T)) : 128, PR = row_b / 16;   // bytes and pieces of a stored row
    static constexpr int Q = row_b < 256 ? 256 / row_b : 1;
    static __device__ __forceinline__ int swizzle(int r) { return COL ? ((r / Q & 3) << 2) & (PR - 1) : r / 2 % 8; }
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
            typedef __attribute__((address_space(3))) s4_t* lds4;
            const int b = (w0 + (lane & 16) + (lane & 3) * 4) * 2, k = c * V + ((lane & 15) >> 2);
            const s4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(s + piece(k, b >> 4) + (b & 15)));
            const s4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(s + piece(k + 4, b >> 4) + (b & 15)));
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

// Rows at any distance and alignment: a tile of BM rows x BN features by WM x WN waves, one stage of LDS, the next stage's operands in registers
// while this one is multiplied.
template <typename T, Mode MODE, bool EIGHT, int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(64 * WM * WN) k_product_any(ProductArgs p, int nx, int ny, FastDiv divx, FastDiv divy) {
    constexpr int NT = 64 * WM * WN, V = Chunk<T>::V, FM = BM / WM / 32, FN = BN / WN / 32;
    constexpr bool XCOL = MODE == kWgrad, YCOL = MODE != kProduct;
    using SX = Stage<T, BM, XCOL>;
    using SY = Stage<T, BN, YCOL>;
    constexpr int PX = BM * 8 / NT, PY = BN * 8 / NT, BK = SX::BK;
    static_assert(BM * 8 % NT == 0 && BN * 8 % NT == 0, "whole pieces per thread");
    __shared__ __align__(16) uint8_t s_x[SX::bytes], s_y[SY::bytes];
    __shared__ int s_row[BM];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
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
        for (int i = tid; i < BM; i += NT) {
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
    f16_t acc[FM][FN];
#pragma unroll
    for (int m = 0; m < FM; ++m)
#pragma unroll
        for (int f = 0; f < FN; ++f)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[m][f][i] = 0.0f;
    if (K > 0) load(0);
    for (int k0 = 0; k0 < K; k0 += BK) {
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
        if (K - k0 > BK) load(k0 + BK);
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

template <typename T, Mode MODE, bool EIGHT, int BM, int BN, int WM, int WN>
static int any_go(const char* what, const ProductArgs& p, hipStream_t stream) {
    const int features = MODE == kProduct ? p.N : p.C, ny = (features + BN - 1) / BN, nx = (p.N + BM - 1) / BM;
    const int64_t units = (MODE == kWgrad ? int64_t(p.E) * nx : tiles_at_most(p.M, p.E, BM, p.bounds != nullptr)) * ny;
    if (units > 0x7ffff000) return set_error(kErrShape, "%s: M=%d N=%d C=%d E=%d", what, p.M, p.N, p.C, p.E);
    launch_timed(what, k_product_any<T, MODE, EIGHT, BM, BN, WM, WN>, wide_grid(uint32_t(units)), dim3(64 * WM * WN), 0, stream, p, nx, ny,
                 FastDiv(uint32_t(nx)), FastDiv(uint32_t(ny)));
    FRT_LAUNCHED(what);
    return kOk;
}

template <typename T>
static int product_t(const ProductArgs& p, hipStream_t stream) {
    return any_go<T, kProduct, false, 64, 64, 2, 2>("moe_product", p, stream);
}
template <typename T>
static int grad_t(const ProductArgs& p, hipStream_t stream) {
    return any_go<T, kGrad, false, 64, 64, 2, 2>("moe_product_grad", p, stream);
}
template <typename T>
static int wgrad_t(const ProductArgs& p, hipStream_t stream) {
    return p.scales ? any_go<T, kWgrad, true, 64, 64, 2, 2>("moe_product_wgrad", p, stream) : any_go<T, kWgrad, false, 64, 64, 2, 2>("moe_product_wgrad", p, stream);
}

int moe_product(int type, const ProductArgs& p, hipStream_t stream) { return FRT_BY_TYPE(type, product_t, p, stream); }
int moe_product_grad(int type, const ProductArgs& p, hipStream_t stream) { return FRT_BY_TYPE(type, grad_t, p, stream); }
int moe_product_wgrad(int type, const ProductArgs& p, hipStream_t stream) { return FRT_BY_TYPE(type, wgrad_t, p, stream); }

}  // namespace frt
