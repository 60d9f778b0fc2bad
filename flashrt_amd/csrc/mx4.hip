// Microscaled 4-bit floats: quantisation, and the grouped product of 4-bit operands on the matrix cores.
//
// Format: each 32 consecutive values of a row share one scale byte b, the power of two 2^(b - 127) (255: NaN), and are e2m1 codes
// (sign, two exponent bits, one mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6). Codes [rows][cols / 2], value 2 j in the low half of
// byte j; scales [rows][cols / 32]. This is the operand format of gfx950's scaled matrix instructions: a lane takes one block
// of 32 codes as 16 bytes and its scale as one byte.
#include "common.hpp"
#include "groups.hpp"
#include "lds_dma.hpp"

#include <algorithm>
#include <type_traits>

#include "../../include/flashrt_moe.h"

namespace frt {

typedef uint32_t u4e4_t __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u4e2_t __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u4e1_t __attribute__((ext_vector_type(4), aligned(1)));
typedef uint32_t u2e2_t __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t u4_t __attribute__((ext_vector_type(4)));
typedef float f4_t __attribute__((ext_vector_type(4)));
typedef float f8_t __attribute__((ext_vector_type(8)));
typedef int i4_t __attribute__((ext_vector_type(4)));
typedef int i8_t __attribute__((ext_vector_type(8)));
typedef float f16_t __attribute__((ext_vector_type(16)));

// Eight values of a row as fp32, loaded at the element's own alignment
__device__ __forceinline__ f8_t load8(const float* p) {
    const u4e4_t a = *reinterpret_cast<const u4e4_t*>(p), b = *reinterpret_cast<const u4e4_t*>(p + 4);
    const f4_t x = __builtin_bit_cast(f4_t, a), y = __builtin_bit_cast(f4_t, b);
    return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
}
template <typename T>
__device__ __forceinline__ f8_t load8(const T* p) {
    typedef T v8 __attribute__((ext_vector_type(8)));
    return __builtin_convertvector(__builtin_bit_cast(v8, *reinterpret_cast<const u4e2_t*>(p)), f8_t);
}
__device__ __forceinline__ void store8(float* p, f8_t v) {
    *reinterpret_cast<u4e4_t*>(p) = __builtin_bit_cast(u4e4_t, __builtin_shufflevector(v, v, 0, 1, 2, 3));
    *reinterpret_cast<u4e4_t*>(p + 4) = __builtin_bit_cast(u4e4_t, __builtin_shufflevector(v, v, 4, 5, 6, 7));
}
template <typename T>
__device__ __forceinline__ void store8(T* p, f8_t v) {
    typedef T v8 __attribute__((ext_vector_type(8)));
    *reinterpret_cast<u4e2_t*>(p) = __builtin_bit_cast(u4e2_t, __builtin_convertvector(v, v8));
}

// The fp32 value of a scale byte (0: the subnormal 2^-127)
__device__ __forceinline__ float scale_value(uint32_t b) {
    return __builtin_bit_cast(float, b == 255u ? 0x7fc00000u : b ? b << 23 : 0x00400000u);
}

// ---------------------------------------------------------------- quantisation
// Four lanes to a block, eight values each. With amax = m 2^k (1 <= m < 2) the scale is 2^(k - 2), so the largest code's
// exponent is amax's; its byte k + 125 is the exponent field of amax less 2, at least 0 (2^-127, all smaller blocks). A value's
// code is x 2^-(k - 2), an exact product, rounded to nearest even by the conversion instruction, at most 6. A block with
// an infinity or a NaN (the exponent field 255 in the largest absolute bits) gets the NaN scale and zero codes. Bound by HBM:
// 20480 x 2560 bf16 25 us, 5.3 TB/s.
template <typename T>
__global__ void __launch_bounds__(256) k_mx4_quantize(const T* __restrict__ x, int64_t ldx, uint32_t pieces, uint32_t per_row, FastDiv div,
                                                      uint32_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;   // (pieces is a multiple of 4: whole quads stay or go)
    if (i >= pieces) return;
    const uint32_t r = div(i);
    const f8_t v = load8(x + r * ldx + (i - r * per_row) * 8);
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float f = v[j];   // (a bit cast of a vector's element by itself takes the first one)
        top = max(top, __builtin_bit_cast(uint32_t, f) & 0x7fffffffu);
    }
    top = max(top, uint32_t(__builtin_amdgcn_mov_dpp(int(top), kDppXor1, 0xF, 0xF, true)));
    top = max(top, uint32_t(__builtin_amdgcn_mov_dpp(int(top), kDppXor2, 0xF, 0xF, true)));
    const bool bad = top >= 0x7f800000u;
    const uint32_t b = bad ? 255u : uint32_t(max(int(top >> 23) - 2, 0));
    const float inv = __builtin_bit_cast(float, (254u - min(b, 252u)) << 23);   // 2^(127 - b)
    uint32_t q = 0;
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[0] * inv, v[1] * inv, 1.0f, 0);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[2] * inv, v[3] * inv, 1.0f, 1);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[4] * inv, v[5] * inv, 1.0f, 2);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[6] * inv, v[7] * inv, 1.0f, 3);
    codes[i] = bad ? 0u : q;
    if ((i & 3) == 0) scales[i >> 2] = uint8_t(b);
}

// Eight codes per lane by the conversion instruction: 20480 x 2560 to bf16 25.5 us, 5.2 TB/s (20 with the codes in the last cache, just
// quantised; in integer operations the VALU bound it at 35).
template <typename T>
__global__ void __launch_bounds__(256) k_mx4_dequantize(const uint32_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                        uint32_t pieces, uint32_t per_row, FastDiv div, T* __restrict__ out, int64_t ldout) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i >= pieces) return;
    const uint32_t r = div(i);
    const uint32_t q = codes[i];
    const float s = scale_value(scales[i >> 2]);
    // (the conversion's own scale is an exponent alone: one here, and an exact product for the block's, NaN and 2^-127 included)
    typedef float f2_t __attribute__((ext_vector_type(2)));
    const f2_t a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.0f, 1);
    const f2_t c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.0f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.0f, 3);
    const f8_t v = {a.x * s, a.y * s, b.x * s, b.y * s, c.x * s, c.y * s, d.x * s, d.y * s};
    store8(out + r * ldout + (i - r * per_row) * 8, v);
}

// Rows of one launch: fewer than 2^31 pieces of 8 values
static int64_t launch_rows(int cols) { return (int64_t(0x7fffff00) / (cols / 8)) > 0 ? int64_t(0x7fffff00) / (cols / 8) : 1; }

template <typename T>
static int quantize_t(const void* x, int64_t ldx, int64_t rows, int cols, void* codes, void* scales, hipStream_t stream) {
    const int64_t most = launch_rows(cols);
    for (int64_t r = 0; r < rows; r += most) {
        const uint32_t pieces = uint32_t((rows - r < most ? rows - r : most) * (cols / 8));
        launch_timed("mx4_quantize", k_mx4_quantize<T>, dim3((pieces + 255) / 256), dim3(256), 0, stream, static_cast<const T*>(x) + r * ldx,
                     ldx, pieces, uint32_t(cols / 8), FastDiv(cols / 8), static_cast<uint32_t*>(codes) + r * (cols / 8),
                     static_cast<uint8_t*>(scales) + r * (cols / 32));
        FRT_LAUNCHED("mx4_quantize");
    }
    return kOk;
}
template <typename T>
static int dequantize_t(const void* codes, const void* scales, int64_t rows, int cols, void* out, int64_t ldout, hipStream_t stream) {
    const int64_t most = launch_rows(cols);
    for (int64_t r = 0; r < rows; r += most) {
        const uint32_t pieces = uint32_t((rows - r < most ? rows - r : most) * (cols / 8));
        launch_timed("mx4_dequantize", k_mx4_dequantize<T>, dim3((pieces + 255) / 256), dim3(256), 0, stream,
                     static_cast<const uint32_t*>(codes) + r * (cols / 8), static_cast<const uint8_t*>(scales) + r * (cols / 32), pieces,
                     uint32_t(cols / 8), FastDiv(cols / 8), static_cast<T*>(out) + r * ldout, ldout);
        FRT_LAUNCHED("mx4_dequantize");
    }
    return kOk;
}

// ---------------------------------------------------------------- the grouped product
struct Mx4Args {
    const uint8_t* aq;
    const uint8_t* as;
    int a_rows;
    const int32_t* rows;
    const uint8_t* wq;
    const uint8_t* ws;
    const int32_t* bounds;
    int E, M, N, C;
    void* out;
    int64_t ldout;
};

// An operand of the matrix instructions: its 16 bytes in the low half of the register tuple
__device__ __forceinline__ i8_t fp4(i4_t v) { return __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1); }

// Few rows: 16 features x 16 rows by KW waves that share the values of a row, straight from global memory into the registers of the
// matrix instructions, all of a wave's loads in flight at once. The weights are the first operand, so that a lane's four results
// are adjacent features of one row. A group of 512 values is 16 blocks: step i multiplies blocks 4 i + l / 16 of lane l's
// feature and row, whose scales are the 16 bytes beside each other; wave w takes the groups w, w + KW, ..., and the blocks behind
// the last whole group go one step at a time. The waves' sums are added in their order. Rows and features past the end are the last one
// again, never stored. Bound by the chain of trips to memory (bounds, then the row's index and the weights, then the activations):
// one token's ten experts (N 1024, C 2048, 11 MB) 7.2 us.
template <typename T, int KW>
__global__ void __launch_bounds__(256) k_mx4_rows(Mx4Args p, int ntile, FastDiv ntiles) {
    constexpr int FW = 4 / KW;   // tiles of a workgroup
    __shared__ f4_t s_sum[4][64];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, j = lane & 15, g = lane >> 4;
    const int kw = wave % KW;
    const uint32_t unit = wide_block() * FW + wave / KW, tile = ntiles(unit);
    const RowTile t = find_tile<16>(p.bounds, p.E, p.M, [&](int total) { return int(tile) < total ? int(tile) : -1; });
    const int f0 = int(unit - tile * ntile) * 16, nb = p.C / 32, ng = nb / 16;
    f4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
    bool ok = false;
    if (t.rows > 0) {   // (uniform over the wave)
        const int r = t.row0 + min(j, t.rows - 1);
        int a = r;
        if (p.rows) a = gld<int>(p.rows + r);   // (under way while the weights' loads are issued)
        const int64_t w = (int64_t(t.g) * p.N + min(f0 + j, p.N - 1)) * nb;
        struct Group {
            i4_t w[4], x[4];
            u4e1_t ws, xs;
        } u, v;
        auto load_w = [&](int q, Group& o) {
#pragma unroll
            for (int i = 0; i < 4; ++i) o.w[i] = gld<i4_t>(p.wq + (w + 16 * q + 4 * i + g) * 16);
            o.ws = gld<u4e1_t>(p.ws + w + 16 * q);
        };
        auto load_x = [&](int q, Group& o, int64_t x) {
#pragma unroll
            for (int i = 0; i < 4; ++i) o.x[i] = gld<i4_t>(p.aq + (x + 16 * q + 4 * i + g) * 16);
            o.xs = gld<u4e1_t>(p.as + x + 16 * q);
        };
        auto mma = [&](const Group& o) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fp4(o.w[i]), fp4(o.x[i]), acc, 4, 4, 0, int(o.ws[i] >> (8 * g)), 0,
                                                                       int(o.xs[i] >> (8 * g)));
        };
        int q = kw;
        if (q < ng) load_w(q, u);
        if (q + KW < ng) load_w(q + KW, v);
        __builtin_amdgcn_sched_barrier(0);
        ok = unsigned(a) < unsigned(p.a_rows);
        const int64_t x = int64_t(ok ? a : 0) * nb;
        if (q < ng) load_x(q, u, x);
        if (q + KW < ng) load_x(q + KW, v, x);
        for (; q < ng; q += 2 * KW) {   // two groups' loads in flight
            mma(u);
            if (q + 2 * KW < ng) {
                load_w(q + 2 * KW, u);
                load_x(q + 2 * KW, u, x);
            }
            if (q + KW < ng) {
                mma(v);
                if (q + 3 * KW < ng) {
                    load_w(q + 3 * KW, v);
                    load_x(q + 3 * KW, v, x);
                }
            }
        }
        for (int b = 16 * ng + 4 * kw; b < nb; b += 4 * KW) {   // the last blocks' steps, over the waves
            const bool in = b + g < nb;
            const i4_t zero = {0, 0, 0, 0};
            const int c = min(b + g, nb - 1);
            const i4_t wv = gld<i4_t>(p.wq + (w + c) * 16), xv = gld<i4_t>(p.aq + (x + c) * 16);
            const int ws = gld<uint8_t>(p.ws + w + c), xs = gld<uint8_t>(p.as + x + c);
            acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fp4(in ? wv : zero), fp4(in ? xv : zero), acc, 4, 4, 0, in ? ws : 127, 0,
                                                                   in ? xs : 127);
        }
    }
    if constexpr (KW > 1) {
        s_sum[wave][lane] = acc;
        __syncthreads();
        if (kw != 0) return;
#pragma unroll
        for (int i = 1; i < KW; ++i) acc += s_sum[wave + i][lane];
    }
    if (j < t.rows) {
        typedef T vec4 __attribute__((ext_vector_type(4)));
        typedef std::conditional_t<sizeof(T) == 4, u4e4_t, u2e2_t> Raw;
        vec4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = T(ok ? acc[i] : 0.0f);
        T* const o = static_cast<T*>(p.out) + (t.row0 + j) * p.ldout + f0 + 4 * g;
        if (f0 + 4 * g + 4 <= p.N) {
            *reinterpret_cast<Raw*>(o) = __builtin_bit_cast(Raw, v);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (f0 + 4 * g + i < p.N) o[i] = v[i];
        }
    }
}

// A wave's LDS accesses before are done before those after, across its lanes (they complete in order)
__device__ __forceinline__ void wave_lds_order() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
    asm volatile("" ::: "memory");
}

constexpr int KB = 8;   // blocks of a row in a stage
template <int BM, int BN, int NW, int ST, int SS>
struct TileShape {
    static constexpr int rows = BM + BN;                // operand rows of a stage, the activations first
    static constexpr int code_b = rows * KB * 16;       // a stage: KB blocks of 32 values of each row
    static constexpr int dr = 64 / KB, sr = 256 / (KB * SS);   // rows of a code load, of a load of SS stages' scales
    // loads per wave and stage, and per wave and group of SS stages; with fewer activation loads than waves, some are made twice
    static constexpr int da = BM < dr * NW ? 1 : BM / (dr * NW), dw = BN / (dr * NW);
    static constexpr int sa = BM < sr * NW ? 1 : BM / (sr * NW), sw = BN / (sr * NW);
    static_assert((BM % (dr * NW) == 0 || (dr * NW) % BM == 0) && BN % (dr * NW) == 0 && (BM % (sr * NW) == 0 || (sr * NW) % BM == 0) &&
                  BN % (sr * NW) == 0, "every wave the same loads");
    static constexpr int scale_b = rows * SS * KB;      // a group's scales
    // The results leave through LDS, each wave its part of a slot, in rows of 128 bytes (64 where those do not fit)
    static constexpr int out_row = NW * 32 * 144 > code_b ? 64 : 128, out_b = 32 * (out_row + 16);
    static_assert(NW * out_b <= code_b, "the results in a slot");
    static constexpr int smem = ST * code_b + 2 * scale_b + BM * 4;
};

// Stores through a buffer descriptor: a lane whose offset lies past its bytes stores nothing, without a branch, so that the number of
// store instructions, which the waits on the loads behind them have to count, is fixed.
typedef __amdgpu_buffer_rsrc_t Buffer;
constexpr uint32_t kNoStore = 0x80000000u;

// BM rows x BN features per tile, `per` feature tiles of one row tile after one another in a workgroup of WM x WN waves, from
// LDS. A stage is KB blocks of 32 values of every operand row, in a ring of ST slots, their codes loaded straight into it; block c of
// row r sits at c ^ (r / 2 % 8), so that the sixteen rows of a read phase take sixteen different columns of the banks.
// The scales go the same way, 2 SS words of each row at a time (side by side: the loads' cost is lines, not bytes): those of SS stages
// where the rows of scales are words (WORDS: a multiple of 128 values), else the aligned words around those of SS - 1 stages, of
// which a lane takes its bytes by a shift (a row's first and last word may reach three bytes past the row, the tensor's too: in the same
// aligned word, and unused; reading the bytes within one by one instead cost 4 to 8% of the calls that have such a word). In step t (0..3) lane half h
// multiplies block 4 h + t of its rows, so that a lane's four scales of a stage are one word and the step picks its byte. Step t +
// 1's operands are read before step t's products, the next stage's first ones before the last step's, past the barrier. The
// stages of the feature tiles form one sequence: the next tile's first stages load while this one's results are written.
//
// What bounds it: with few rows to a group the weights' stream (2030 rows over 512 experts, N 1024, C 2048: 68 us, 7.3 TB/s of
// weights); with tens of rows what a CU's loads bring in from beyond L2, about 30 bytes per ns (20480 rows 124 us, 0.57 GB of weights
// and as much again of activations and results; the matrix cores 16% busy); with one large group the matrix cores, 43% busy at the 1.98
// GHz that the card keeps under them, and LDS: a stage's reads and direct loads are 256 KB, at 128 bytes a clock the products' own 2048
// clocks, and two slots with a barrier per stage overlap the two in part (8192 rows, N 8192, C 4096: 149 us, 3.7 PFLOP/s). Measured
// without gain: stages of 128 values with twice the slots (20480 rows 139 -> 158 us), eight waves for the smaller tiles, another first
// stage in each workgroup. The 256-row tile spills 3 VGPRs with scales at any byte, and 1 and 6 SGPRs with fp32 results and whole words.
template <typename T, int BM, int BN, int WM, int WN, int ST, int SS, int PT, bool WORDS>
__global__ void __launch_bounds__(64 * WM * WN) k_mx4_tiles(Mx4Args p, int ntile, int per, FastDiv chunks, uint32_t nchunk, int stream) {
    constexpr int NW = WM * WN;
    using Sh = TileShape<BM, BN, NW, ST, SS>;
    static_assert(SS >= 2 && (ST == 2 || ST == 3) && PT <= 3, "whole words of scales; the waits; the steps before a stage's end");
    constexpr int GS = WORDS ? SS : SS - 1;   // the stages of a group of scales
    constexpr int FM = BM / WM / 32, FN = BN / WN / 32, DA = Sh::da, DW = Sh::dw, D = DA + DW;
    extern __shared__ __align__(16) uint8_t smem[];
    uint8_t* const s_scale = smem + ST * Sh::code_b;
    int32_t* const s_row = reinterpret_cast<int32_t*>(s_scale + 2 * Sh::scale_b);   // [BM]: the activations' row, -1: none
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int lr = lane & 31, h = lane >> 5;
    // Workgroup b runs on XCD b % 8. Each XCD takes an eighth of the row tiles, neighbours, with all their features: a tile's activations
    // and, where a group has several tiles, its weights stay in one L2. Where eighths would leave more than a ninth of the chip
    // idle, the workgroups of a tile are neighbours instead.
    uint32_t jt = chunks(blockIdx.x >> 3), chunk = (blockIdx.x >> 3) - jt * nchunk;
    const RowTile t = find_tile<BM>(p.bounds, p.E, p.M, [&](int total) {
        const int each = (total + 7) / 8;
        if (each * 8 - total > total / 8) {
            jt = chunks(blockIdx.x);
            chunk = blockIdx.x - jt * nchunk;
            return int(jt) < total ? int(jt) : -1;
        }
        const int index = int(blockIdx.x & 7) * each + int(jt);
        return int(jt) < each && index < total ? index : -1;
    });
    if (t.rows == 0) return;
    const int nb = p.C / 32, nst = (nb + KB - 1) / KB, nfull = nb / KB;
    int ft = int(chunk) * per;   // this feature tile, and the end
    const int ft1 = min(ft + per, ntile);
    if (tid < BM) {
        const int r = t.row0 + min(tid, t.rows - 1);
        const int a = p.rows ? p.rows[r] : r;
        s_row[tid] = unsigned(a) < unsigned(p.a_rows) ? a : -1;
    }
    __syncthreads();

    // Operand rows past the group's rows and the features are the last one again (never stored). s_row is read here only: a read of
    // LDS behind the direct loads would wait for them all.
    const int am = (wave / WN) * FM * 32 + lr, wf = BM + (wave % WN) * FN * 32 + lr;   // the lane's first stage rows
    uint32_t none = 0;   // bit m: the lane's row 32 m on has no activations
#pragma unroll
    for (int m = 0; m < FM; ++m) none |= uint32_t(s_row[am + 32 * m] < 0) << m;
    const uint8_t* const wq = p.wq + int64_t(t.g) * p.N * nb * 16;
    const uint8_t* const ws = p.ws + int64_t(t.g) * p.N * nb;
    auto wgt_row = [&](int f, int r) { return int64_t(min(f * BN + r, p.N - 1)) * nb; };   // the first scale of row r of feature tile f
    // codes: a wave loads DA dr rows of activations and DW dr of weights; the next stage to load is stage jst of feature tile jf, into
    // slot jslot
    constexpr int dr = Sh::dr;
    const uint8_t* asrc[DA];
    const uint8_t* wsrc[DW];
    const int aw = wave * DA % (BM / dr), ww = wave * DW;   // the wave's first loads
#pragma unroll
    for (int i = 0; i < DA; ++i) asrc[i] = p.aq + int64_t(max(s_row[(aw + i) * dr + lane / KB], 0)) * nb * 16;
    int jf = ft, jst = 0, jslot = 0;
    auto point = [&]() {
#pragma unroll
        for (int i = 0; i < DW; ++i) wsrc[i] = wq + wgt_row(jf, (ww + i) * dr + lane / KB) * 16;
    };
    // Weights that no other row tile reads, in whole lines, are streamed past the activations in L2: 2048 rows over 512 experts (N
    // 1024, C 2048) 78 -> 70 us, 20480 even ones 126 -> 115. Rows that share lines (C 640) would be fetched again: 75 -> 90.
    const bool once = stream && t.only && nb % 8 == 0;
    // Part k of PT of that stage's loads (blocks past the row's last read as its last: their steps are masked); the last part moves on
    auto column = [&](int r) { return (lane % KB) ^ ((r + lane / KB) / (16 / KB) % KB); };   // the block at the lane's place in a load from row r on
    auto issue_part = [&](auto kc) {
        constexpr int k = decltype(kc)::value;
        if (jf >= ft1) return;
        uint8_t* const s = smem + jslot * Sh::code_b;
#pragma unroll
        for (int i = DA * k / PT; i < DA * (k + 1) / PT; ++i)
            ldsdma16(asrc[i] + min(KB * jst + column((aw + i) * dr), nb - 1) * 16, s + (aw + i) * 1024);
        if (once) {
#pragma unroll
            for (int i = DW * k / PT; i < DW * (k + 1) / PT; ++i)
                ldsdma16_nt(wsrc[i] + min(KB * jst + column((ww + i) * dr), nb - 1) * 16, s + BM * KB * 16 + (ww + i) * 1024);
        } else {
#pragma unroll
            for (int i = DW * k / PT; i < DW * (k + 1) / PT; ++i)
                ldsdma16(wsrc[i] + min(KB * jst + column((ww + i) * dr), nb - 1) * 16, s + BM * KB * 16 + (ww + i) * 1024);
        }
        if (k < PT - 1) return;
        jslot = jslot == ST - 1 ? 0 : jslot + 1;
        if (++jst == nst) {
            jst = 0;
            ++jf;
            point();
        }
    };
    auto issue = [&]() {
        issue_part(std::integral_constant<int, 0>());
        if constexpr (PT > 1) issue_part(std::integral_constant<int, 1>());
        if constexpr (PT > 2) issue_part(std::integral_constant<int, 2>());
    };
    bool parts = false;   // parts 1 .. of a stage's loads are still to be issued
    auto issue_more = [&](auto kc) {
        constexpr int k = decltype(kc)::value;
        if constexpr (k < PT) {
            if (parts) issue_part(kc);
        }
    };
    // scales: the next group is that of stages sq GS .. of feature tile sf, into buffer sbuf
    constexpr int LR = KB * SS / 4;   // lanes (words) of a row's group
    constexpr int NA = Sh::sa, NS = Sh::sa + Sh::sw;   // the first NA are the activations'
    const uint8_t* ssrc[NS];
    int sf = ft, sq = 0, sbuf = 0;
    const int sw0 = wave * Sh::sa % (BM / Sh::sr > 0 ? BM / Sh::sr : 1);   // the wave's first load of the activations'
#pragma unroll
    for (int k = 0; k < NA; ++k) ssrc[k] = p.as + int64_t(max(s_row[(sw0 + k) * Sh::sr + lane / LR], 0)) * nb;
    auto spoint = [&]() {
#pragma unroll
        for (int k = NA; k < NS; ++k) ssrc[k] = ws + wgt_row(sf, (wave * Sh::sw + k - NA) * Sh::sr + lane / LR);
    };
    auto byte_of = [](const uint8_t* q) { return WORDS ? 0 : int(reinterpret_cast<uintptr_t>(q) & 3); };   // in its word
    auto issue_scales = [&]() {
        if (sf >= ft1) return;
        uint8_t* const s = s_scale + sbuf * Sh::scale_b;
#pragma unroll
        for (int k = 0; k < NS; ++k) {   // (words past the row's end read as its last)
            const int off = byte_of(ssrc[k]), w = min(2 * GS * sq + lane % LR, (off + nb - 1) / 4) * 4 - off;
            ldsdma4(ssrc[k] + w, s + (k < NA ? (sw0 + k) * 256 : BM * SS * KB + (wave * Sh::sw + k - NA) * 256));
        }
        sbuf ^= 1;
        if (++sq * GS >= nst) {
            sq = 0;
            ++sf;
            spoint();
        }
    };
    // The first byte of the lane's rows' scales (the weights' rows are a multiple of 32 apart, over the feature tiles too; of a row past
    // the last feature the bytes are another's, and not used)
    int a_off[FM];
#pragma unroll
    for (int m = 0; m < FM; ++m) a_off[m] = byte_of(p.as + int64_t(max(s_row[am + 32 * m], 0)) * nb);
    const int w_off = byte_of(ws + int64_t(wf - BM) * nb);
    point();
    spoint();
    issue_scales();
    issue_scales();
#pragma unroll
    for (int s = 0; s < ST; ++s) issue();

    const int sw = lr / (16 / KB) % KB;   // (of all its rows: they are 32 apart)
    struct Ops {
        i4_t a[FM], b[FN];
    };
    auto read = [&](int slot, int tt) {
        const uint8_t* const s = smem + slot * Sh::code_b + ((KB / 2 * h + tt) ^ sw) * 16;
        Ops o;
#pragma unroll
        for (int m = 0; m < FM; ++m) o.a[m] = *reinterpret_cast<const i4_t*>(s + (am + 32 * m) * KB * 16);
#pragma unroll
        for (int f = 0; f < FN; ++f) o.b[f] = *reinterpret_cast<const i4_t*>(s + (wf + 32 * f) * KB * 16);
        return o;
    };
    struct Scales {
        int a[FM], b[FN];
    };
    auto read_scales = [&](int st, int buf) {
        const uint8_t* const s = s_scale + buf * Sh::scale_b + (st % GS) * KB + h * 4;
        auto four = [&](int row, int off) {
            const int* const w = reinterpret_cast<const int*>(s + row * KB * SS);
            return WORDS ? w[0] : int(__builtin_amdgcn_alignbyte(w[1], w[0], off));
        };
        Scales o;
#pragma unroll
        for (int m = 0; m < FM; ++m) o.a[m] = four(am + 32 * m, a_off[m]);
#pragma unroll
        for (int f = 0; f < FN; ++f) o.b[f] = four(wf + 32 * f, w_off);
        return o;
    };
    f16_t acc[FM][FN];
    auto mma = [&](auto tc, const Ops& o, const Scales& s) {   // (features x rows: a lane's four results in a row are adjacent features)
        constexpr int tt = decltype(tc)::value;
#pragma unroll
        for (int m = 0; m < FM; ++m)
#pragma unroll
            for (int f = 0; f < FN; ++f)
                acc[m][f] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fp4(o.b[f]), fp4(o.a[m]), acc[m][f], 4, 4, tt, s.b[f], tt, s.a[m]);
    };
    auto pin = [&]() {   // the products before stay before what follows (else the compiler sinks them past the barrier)
#pragma unroll
        for (int m = 0; m < FM; ++m)
#pragma unroll
            for (int f = 0; f < FN; ++f) asm volatile("" : "+a"(acc[m][f]));
    };

    // Waits count the codes' loads: at the end of a stage those of `under` (ST - 1, fewer at the sequence's end) stages after it have
    // been issued last, the next one's first. In a feature tile's first stages the stores of the tile before (kStores per wave)
    // came behind the loads that are waited for, and may be under way too.
    constexpr int kStores = FM * FN * int(sizeof(T)), kAfter = D * (ST - 2) + kStores;
    const int ft0 = ft;
    int under = min(ST, (ft1 - ft) * nst) - 1;
    if ((ft1 - ft) * nst >= ST)
        wait_vm<D*(ST - 1)>();
    else
        wait_vm<0>();
    ring_barrier();
    int slot = 0, buf = 0;   // the stage being multiplied, and its scales
    Ops o0 = read(0, 0);
    Scales sc = read_scales(0, 0);
    lds_reads_done();   // (nothing pending where the loop is entered: its waits are then for its own reads)
    for (; ft < ft1; ++ft) {
#pragma unroll
        for (int m = 0; m < FM; ++m)
#pragma unroll
            for (int f = 0; f < FN; ++f)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[m][f][i] = 0.0f;
        // the end of stage st: the next stage has landed, all waves have read this one; its slot and, past a group, its scales' buffer
        // are loaded anew (the slot of a tile's last stage after its results were written through it)
        auto finish = [&](int st) {
            const bool last = st + 1 == nst, turn = last || (st + 1) % GS == 0;
            const int nbuf = turn ? buf ^ 1 : buf;
            if (under == ST - 1) {
                if (st < ST - 2 && ft > ft0)
                    wait_vm<(kAfter < 63 ? kAfter : 63)>();
                else
                    wait_vm<D*(ST - 2)>();
            } else {
                wait_vm<0>();
            }
            if (jf >= ft1) --under;
            ring_barrier();
            if (turn) issue_scales();
            parts = PT > 1 && !last;
            if (parts)
                issue_part(std::integral_constant<int, 0>());
            else if (!last)
                issue();
            buf = nbuf;
            slot = slot == ST - 1 ? 0 : slot + 1;
        };
        for (int st = 0; st < nfull; ++st) {
            Ops o1 = read(slot, 1);
            issue_more(std::integral_constant<int, 1>());
            __builtin_amdgcn_sched_barrier(0);
            mma(std::integral_constant<int, 0>(), o0, sc);
            if constexpr (PT > 1) pin();
            __builtin_amdgcn_sched_barrier(0);
            const Ops o2 = read(slot, 2);
            issue_more(std::integral_constant<int, 2>());
            __builtin_amdgcn_sched_barrier(0);
            mma(std::integral_constant<int, 1>(), o1, sc);
            if constexpr (PT > 1) pin();
            __builtin_amdgcn_sched_barrier(0);
            o1 = read(slot, 3);
            __builtin_amdgcn_sched_barrier(0);
            mma(std::integral_constant<int, 2>(), o2, sc);
            pin();
            finish(st);
            o0 = read(slot, 0);   // (past the last stage: nothing that is used)
            const Scales next = read_scales(st + 1 == nst ? 0 : st + 1, buf);
            __builtin_amdgcn_sched_barrier(0);
            mma(std::integral_constant<int, 3>(), o1, sc);
            sc = next;
        }
        if (nfull < nst) {
            // the last, shorter stage: blocks 2 i and 2 i + 1 in step i; a block past the row's end is zeros at scale one
            issue_more(std::integral_constant<int, 1>());
            issue_more(std::integral_constant<int, 2>());
            const uint8_t* const s = smem + slot * Sh::code_b;
            const uint8_t* const ssc = s_scale + buf * Sh::scale_b + (nfull % GS) * KB;
            const int left = nb - KB * nfull;
            const i4_t zero = {0, 0, 0, 0};
            for (int c = h; c - h < left; c += 2) {
                const bool in = c < left;
                const int at = (c ^ sw) * 16;
                i4_t b[FN];
                int bs[FN];
#pragma unroll
                for (int f = 0; f < FN; ++f) {
                    b[f] = *reinterpret_cast<const i4_t*>(s + (wf + 32 * f) * KB * 16 + at);
                    bs[f] = ssc[(wf + 32 * f) * KB * SS + w_off + c];
                    b[f] = in ? b[f] : zero;
                    bs[f] = in ? bs[f] : 127;
                }
#pragma unroll
                for (int m = 0; m < FM; ++m) {
                    i4_t a = *reinterpret_cast<const i4_t*>(s + (am + 32 * m) * KB * 16 + at);
                    int as = ssc[(am + 32 * m) * KB * SS + a_off[m] + c];
                    a = in ? a : zero;
                    as = in ? as : 127;
#pragma unroll
                    for (int f = 0; f < FN; ++f)
                        acc[m][f] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fp4(b[f]), fp4(a), acc[m][f], 4, 4, 0, bs[f], 0, as);
                }
            }
            finish(nfull);
            o0 = read(slot, 0);
            sc = read_scales(0, buf);
        }

        // The results through LDS, 32 rows of QP fourths of a fragment (8 features each) at a time, so that whole lines are stored.
        // Lane l's value i of a fragment: feature 8 (i / 4) + 4 h + i % 4, row l % 32.
        constexpr int sz = sizeof(T), QP = Sh::out_row / (8 * sz) < 4 * FN ? Sh::out_row / (8 * sz) : 4 * FN, V = 16 / sz;
        constexpr int PR = QP * 8 / V, NP = 32 * PR / 64, RS = Sh::out_row + 16;   // pieces of 16 bytes in a row, of a lane; bytes from row to row
        static_assert(4 * FN % QP == 0 && FM * (4 * FN / QP) * NP == kStores, "the stores of a wave");
        typedef T vec4 __attribute__((ext_vector_type(4)));
        uint8_t* const w = smem + (slot == 0 ? ST - 1 : slot - 1) * Sh::code_b + wave * (Sh::code_b / NW);
        T* const out = static_cast<T*>(p.out) + t.row0 * p.ldout;
        const Buffer buffer = __builtin_amdgcn_make_buffer_rsrc(out, 0, int(((t.rows - 1) * p.ldout + p.N) * sz), 0x00020000);
#pragma unroll
        for (int m = 0; m < FM; ++m) {
            const bool ok = !(none >> m & 1);
#pragma unroll
            for (int q = 0; q < 4 * FN; q += QP) {
#pragma unroll
                for (int g = q / 4; g <= (q + QP - 1) / 4; ++g) asm volatile("" : "+a"(acc[m][g]));   // (read one piece at a time)
#pragma unroll
                for (int i = 0; i < QP; ++i) {
                    vec4 v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = T(ok ? acc[m][(q + i) / 4][(q + i) % 4 * 4 + e] : 0.0f);
                    *reinterpret_cast<vec4*>(w + lr * RS + (8 * i + 4 * h) * sz) = v;
                }
                wave_lds_order();
                int ln = lane;
                asm volatile("" : "+v"(ln));   // (addresses formed piece by piece, not all kept from before the loop)
                const int at = ft * BN + (wave % WN) * FN * 32 + q * 8 + ln % PR * V;
                const int r0 = (wave / WN) * FM * 32 + 32 * m + ln / PR;
                const uint8_t* const l = w + ln / PR * RS + ln % PR * 16;
                if ((ft + 1) * BN <= p.N) {
                    i4_t v[NP];
#pragma unroll
                    for (int i = 0; i < NP; ++i) v[i] = *reinterpret_cast<const i4_t*>(l + i * (64 / PR) * RS);
#pragma unroll
                    for (int i = 0; i < NP; ++i) {
                        const int r = r0 + i * (64 / PR);
                        const uint32_t to = r < t.rows ? uint32_t(r * int(p.ldout) + at) * sz : kNoStore;
                        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4_t, v[i]), buffer, to, 0, 2);   // (non-temporal)
                    }
                } else {   // the last feature tile, cut short
                    for (int i = 0; i < NP && r0 + i * (64 / PR) < t.rows; ++i)
                        for (int e = 0; e < V && at + e < p.N; ++e)
                            out[(r0 + i * (64 / PR)) * p.ldout + at + e] = *reinterpret_cast<const T*>(l + i * (64 / PR) * RS + e * sz);
                }
                wave_lds_order();
            }
        }
        ring_barrier();   // every wave's results have left the slot
        issue();
    }
}

template <typename T, int BM, int BN, int WM, int WN, int ST, int SS, int PT, bool WORDS>
static int tiles_go(const Mx4Args& p, int stages, int64_t fill, hipStream_t stream) {
    const int ntile = (p.N + BN - 1) / BN;
    const int64_t tiles = tiles_at_most(p.M, p.E, BM, p.bounds != nullptr);
    // feature tiles of a workgroup: about `stages` stages, as long as `fill` workgroups remain (half a tile of each group empty)
    const int nst = (p.C / 32 + 7) / 8;
    const int64_t groups = std::min(p.E, p.M), likely = p.bounds ? std::max<int64_t>(p.M / BM + groups / 2, groups) : tiles;
    int nchunk = std::max(1, std::min(stages / nst, ntile));
    nchunk = (ntile + nchunk - 1) / nchunk;
    while (nchunk < ntile && likely * nchunk < fill) ++nchunk;
    const int per = (ntile + nchunk - 1) / nchunk;
    nchunk = (ntile + per - 1) / per;
    // (few rows to a group: only weights beyond the 256 MB of the last cache; 80 experts, 84 MB, read again and again 15.2 against 21.1 us)
    const int stream_w = BM > 32 || groups * p.N * (p.C / 2) > (int64_t(256) << 20);
    const int64_t wgs = (tiles + 7) / 8 * 8 * nchunk;
    if (wgs * (64 * WM * WN) > 0xffffffff) return set_error(kErrShape, "mx4_product: M=%d N=%d E=%d", p.M, p.N, p.E);   // (the launch's threads)
    constexpr int smem = TileShape<BM, BN, WM * WN, ST, SS>::smem;
    static_assert(smem <= 160 * 1024, "LDS of a CU");
    FRT_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(&k_mx4_tiles<T, BM, BN, WM, WN, ST, SS, PT, WORDS>),
                                hipFuncAttributeMaxDynamicSharedMemorySize, smem));
    launch_timed("mx4_product", k_mx4_tiles<T, BM, BN, WM, WN, ST, SS, PT, WORDS>, dim3(uint32_t(wgs)), dim3(64 * WM * WN), smem, stream, p, ntile,
                 per, FastDiv(nchunk), uint32_t(nchunk), stream_w);
    FRT_LAUNCHED("mx4_product");
    return kOk;
}
template <typename T, int BM, int BN, int WM, int WN, int ST, int SS, int PT>
static int tiles_t(const Mx4Args& p, int stages, int64_t fill, hipStream_t stream) {
    const bool words = p.C % 128 == 0 && reinterpret_cast<uintptr_t>(p.as) % 4 == 0 && reinterpret_cast<uintptr_t>(p.ws) % 4 == 0;
    // (20480 rows, N 1000, C 1056: 112 us; through registers, which wait for all loads, 119)
    return words ? tiles_go<T, BM, BN, WM, WN, ST, SS, PT, true>(p, stages, fill, stream)
                 : tiles_go<T, BM, BN, WM, WN, ST, SS, PT, false>(p, stages, fill, stream);
}

template <typename T, int KW>
static int rows_t(const Mx4Args& p, hipStream_t stream) {
    const int ntile = (p.N + 15) / 16;
    const int64_t units = tiles_at_most(p.M, p.E, 16, p.bounds != nullptr) * ntile, wgs = (units + 4 / KW - 1) / (4 / KW);
    if (units > 0x7ffff000) return set_error(kErrShape, "mx4_product: M=%d N=%d E=%d", p.M, p.N, p.E);
    launch_timed("mx4_product", k_mx4_rows<T, KW>, wide_grid(uint32_t(wgs)), dim3(256), 0, stream, p, ntile, FastDiv(ntile));
    FRT_LAUNCHED("mx4_product");
    return kOk;
}

template <typename T>
static int product_t(const Mx4Args& p, hipStream_t stream) {
    // The kernel by the rows of a group, were they spread evenly. With few rows the weights' bytes are all there is to read, and small
    // tiles put more of them in flight; with many the operands pass through LDS less often. us, smaller against larger:
    //   values split over the waves / tiles of 32, by the weights that tiles of 16 rows read: one token's ten experts (N 1024, C 2048,
    //     10 MB) 7.2 / 7.8, two tokens' 11.2 / 9.4, one group (N 8192, C 4096) of 16 rows (16 MB) 8.4 / 12.4, of 24 13.3 / 12.5
    //   32 / 64 (512 experts, N 1024, C 2048): 4 rows to an expert 68 / 74, 16 rows 108 / 107, 40 rows 143 / 123
    //   64 / 128: 40 rows 123 / 149, 62 rows 147 / 140, 160 rows 264 / 240; one group of 512 (N, C 2560) 10.3 / 12.1
    //   128 / 256: 160 rows 240 / 276; 16 experts (N, C 2048) of 300 rows 24.3 / 23.1, 8 of 512 23.4 / 21.5; one group of 8192 (N 8192,
    //     C 4096) 201 / 149
    const int64_t groups = p.bounds ? std::min(p.E, p.M) : 1, avg = p.M / groups;
    auto rows = [&](int64_t BM) { return (avg + BM - 1) / BM * groups; };   // tiles of BM rows
    auto tiles = [&](int64_t BM, int64_t BN) { return rows(BM) * ((p.N + BN - 1) / BN); };
    const int nb = p.C / 32;   // (the tile kernels store through 31-bit offsets)
    if (rows(16) * p.N * (p.C / 2) > (int64_t(16) << 20) && int64_t(256) * p.ldout * int64_t(sizeof(T)) < 0x7fffffff) {
        if (avg >= 256 && tiles(256, 256) >= 128) return tiles_t<T, 256, 256, 4, 2, 2, 2, 3>(p, 64, 256, stream);
        if (avg > 56 && tiles(128, 128) >= 256) return tiles_t<T, 128, 128, 2, 2, 2, 2, 1>(p, 32, 1536, stream);
        if (avg > 8 && tiles(64, 128) >= 160) return tiles_t<T, 64, 128, 2, 2, 3, 2, 1>(p, 16, 512, stream);
        return tiles_t<T, 32, 128, 1, 4, 2, 4, 1>(p, 16, 512, stream);
    }
    return nb >= 64 ? rows_t<T, 4>(p, stream) : nb >= 32 ? rows_t<T, 2>(p, stream) : rows_t<T, 1>(p, stream);
}

int mx4_quantize(int type, const void* x, int64_t ldx, int64_t rows, int cols, void* codes, void* scales, hipStream_t stream) {
    return FRT_BY_TYPE(type, quantize_t, x, ldx, rows, cols, codes, scales, stream);
}
int mx4_dequantize(int type, const void* codes, const void* scales, int64_t rows, int cols, void* out, int64_t ldout,
                   hipStream_t stream) {
    return FRT_BY_TYPE(type, dequantize_t, codes, scales, rows, cols, out, ldout, stream);
}
int mx4_product(const void* aq, const void* as, int a_rows, const int32_t* rows, const void* wq, const void* ws, const int32_t* bounds,
                int E, int M, int N, int C, void* out, int type, int64_t ldout, hipStream_t stream) {
    const Mx4Args p{static_cast<const uint8_t*>(aq), static_cast<const uint8_t*>(as), a_rows, rows, static_cast<const uint8_t*>(wq),
                    static_cast<const uint8_t*>(ws), bounds, E, M, N, C, out, ldout};
    return FRT_BY_TYPE(type, product_t, p, stream);
}

}  // namespace frt
