// Microscaled 4-bit floating point (e2m1 values, one power-of-two scale for each 32 values of a row): packing, unpacking, and the
// linear layer y = x w^T + bias with both operands in that form on the scaled matrix instructions.
//
//     e = floor(log2(max |x| of the 32 values)) - 2,   code = e2m1(x / 2^e), nearest, ties to even, beyond 6 -> 6
// The scale is stored as the byte e + 127 (e >= -127; all-zero blocks get 0); a NaN or an infinity among the 32 makes it 255, which
// stands for NaN.  Rows are padded with zeros to whole slices of 128 values:
//     codes  [rows][slices][64 bytes], two codes a byte, the even column in the low half
//     scales [slices][rows][4 bytes]: the four scales of a row's slice are one dword, and those of neighbouring rows are
//            neighbours, so a tile of rows gets its scales with coalesced loads
#include "common.h"
#include <atomic>
#include <type_traits>

namespace segk {

constexpr int kSlice = 128;
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// n / d for n < 2^31 by a multiplication (d fixed on the host)
struct Divide {
    uint32_t d, magic, shift;
    explicit Divide(uint32_t d_) : d(d_) {
        uint32_t l = 0;
        while ((1ull << l) < d) ++l;
        shift = 31 + l;
        magic = (uint32_t)(((1ull << shift) + d - 1) / d);
    }
    __device__ __forceinline__ uint32_t operator()(uint32_t n) const { return (uint32_t)(((uint64_t)n * magic) >> shift); }
};

// 16 bytes from an address that is only aligned to its elements
template <typename T> struct alignas(sizeof(T)) Raw16 { T e[16 / sizeof(T)]; };

template <typename T> __device__ __forceinline__ void load8_any(const T* p, float (&v)[8]) {
    constexpr int N = 16 / (int)sizeof(T);
#pragma unroll
    for (int h = 0; h < 8 / N; ++h) {
        Raw16<T> r;
        __builtin_memcpy(&r, p + h * N, 16);
#pragma unroll
        for (int i = 0; i < N; ++i) v[h * N + i] = Elem<T>::to_f(r.e[i]);
    }
}
template <typename T> __device__ __forceinline__ void store8_any(T* p, const float (&v)[8]) {
    constexpr int N = 16 / (int)sizeof(T);
#pragma unroll
    for (int h = 0; h < 8 / N; ++h) {
        Raw16<T> r;
#pragma unroll
        for (int i = 0; i < N; ++i) r.e[i] = Elem<T>::from_f(v[h * N + i]);
        __builtin_memcpy(p + h * N, &r, 16);
    }
}

// The scale byte of a block from the bits of its largest magnitude, and the factor that divides by the scale.  The exponent field
// of a float is floor(log2) + 127, so the byte is that field less 2; fields up to 2 (and subnormals) give the smallest scale.
__device__ __forceinline__ uint32_t scale_byte(uint32_t top) {
    const uint32_t f = top >> 23;
    return f == 255u ? 255u : (f > 2u ? f - 2u : 0u);
}
__device__ __forceinline__ float scale_inverse(uint32_t byte) { return byte == 255u ? 0.f : __uint_as_float((254u - byte) << 23); }
__device__ __forceinline__ float scale_value(uint32_t byte) {
    return __uint_as_float(byte == 255u ? 0x7FC00000u : byte == 0u ? 0x00400000u : byte << 23);
}
// eight values, already divided by their scale, as eight codes
__device__ __forceinline__ uint32_t pack_codes(const float (&y)[8]) {
    uint32_t r = 0;
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, y[0], y[1], 1.f, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, y[2], y[3], 1.f, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, y[4], y[5], 1.f, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, y[6], y[7], 1.f, 3);
    return r;
}
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
    uint32_t o = (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true);      // lane ^ 1
    v = v > o ? v : o;
    o = (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, true);               // lane ^ 2
    return v > o ? v : o;
}

// The codes of values c0 .. c0 + 7 of a row (zeros beyond its end) and the scale byte of their block; the four lanes of a block, which
// are neighbours, have to call it together.
template <typename T> __device__ __forceinline__ uint32_t pack_eight(const T* __restrict__ row, int c0, int cols, uint32_t& byte) {
    float v[8];
    const T* p = row + c0;
    if (c0 + 8 <= cols) load8_any<T>(p, v);
    else
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = c0 + j < cols ? Elem<T>::to_f(p[j]) : 0.f;
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t b = __float_as_uint(v[j]) & 0x7FFFFFFFu;
        top = top > b ? top : b;
    }
    byte = scale_byte(quad_max(top));
    const float inv = scale_inverse(byte);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = byte == 255u ? 0.f : v[j] * inv;
    return pack_codes(v);
}

// One thread for 8 values, four neighbouring threads for a block, sixteen for a slice of a row: 16 bytes (bf16) read and 4 written
// per thread, both coalesced.  Bound by memory: 8192 x 8192 bf16 (134 MB read, 36 written) 31 us, 5.5 TB/s; unpacking them again
// 31 us.
template <typename T>
__global__ __launch_bounds__(256) void mxfp4_quantize_kernel(const T* __restrict__ x, int64_t ld, int cols, uint32_t items, Divide per_row,
                                                             int64_t scale_rows, int64_t row0, uint32_t* __restrict__ codes,
                                                             uint32_t* __restrict__ scales) {
    const uint32_t item = blockIdx.x * 256u + threadIdx.x;
    if (item >= items) return;                                     // items are whole slices: a group of 16 lanes leaves together
    const uint32_t r = per_row(item), i = item - r * per_row.d;
    const int64_t row = row0 + r;
    const int c0 = (int)i * 8;
    uint32_t byte;
    codes[row * per_row.d + i] = pack_eight<T>(x + row * ld, c0, cols, byte);
    const int lane = threadIdx.x & 63;
    const uint32_t b1 = __shfl(byte, (lane & 48) + 4, 64), b2 = __shfl(byte, (lane & 48) + 8, 64), b3 = __shfl(byte, (lane & 48) + 12, 64);
    if ((i & 15u) == 0) scales[(int64_t)(i >> 4) * scale_rows + row] = byte | (b1 << 8) | (b2 << 16) | (b3 << 24);
}

template <typename T>
__global__ __launch_bounds__(256) void mxfp4_dequantize_kernel(const uint32_t* __restrict__ codes, const uint8_t* __restrict__ scales, int cols,
                                                               uint32_t items, Divide per_row, int64_t rows, int64_t row0, T* __restrict__ y,
                                                               int64_t ld) {
    const uint32_t item = blockIdx.x * 256u + threadIdx.x;
    if (item >= items) return;
    const uint32_t r = per_row(item), i = item - r * per_row.d;
    const int64_t row = row0 + r;
    const int c0 = (int)i * 8;
    if (c0 >= cols) return;
    const uint32_t c = codes[row * per_row.d + i];
    const float s = scale_value(scales[((int64_t)(i >> 4) * rows + row) * 4 + ((i >> 2) & 3)]);
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        // the magnitude 0, .5, 1, 1.5, 2, 3, 4, 6 as a float: two exponent bits and one fraction bit moved to their places
        const uint32_t m = (c >> (4 * j)) & 7u;
        const float f = m < 2u ? 0.5f * (float)m : __uint_as_float(((m >> 1) + 126u) << 23 | (m & 1u) << 22);
        v[j] = __uint_as_float(__float_as_uint(f * s) | ((c >> (4 * j)) & 8u) << 28);
    }
    T* p = y + row * ld + c0;
    if (c0 + 8 <= cols) store8_any<T>(p, v);
    else
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (c0 + j < cols) p[j] = Elem<T>::from_f(v[j]);
}

// ------------------------------------------------------------------------------------------------ the product
__device__ __forceinline__ f32x4 mfma_fp4(const u32x4 a, const u32x4 b, const f32x4 acc, uint32_t sa, uint32_t sb) {
    const i32x8 av = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0}, bv = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, acc, 4, 4, 0, (int)sa, 0, (int)sb);
}

struct LinearArgs {
    const uint8_t* w;            // codes of the weights [N][ldc]
    const uint32_t* ws;          // their scales [slices][N]
    const uint8_t* x;            // codes of the inputs [M][ldc]
    const uint32_t* xs;
    const float* bias;
    void* y;
    int64_t M, N, ldc, ldy, xs_rows;      // xs_rows: rows from one slice to the next in xs
    int slices, vec;             // vec: so many neighbouring outputs, from a column that is a multiple of it, may be stored at once (0: one)
};

template <typename TO>
__device__ __forceinline__ void store_outputs(const LinearArgs& a, int64_t m, int64_t n, const f32x4 acc) {
    if (m >= a.M || n >= a.N) return;
    TO* y = static_cast<TO*>(a.y) + m * a.ldy + n;
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = acc[i] + (a.bias && n + i < a.N ? a.bias[n + i] : 0.f);
    if (a.vec && n + 4 <= a.N) Elem<TO>::store4(y, v);
    else
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (n + i < a.N) y[i] = Elem<TO>::from_f(v[i]);
}

// Row m of a wave's tile: lane group q holds outputs n + i*16 + 4q .. +3 for the TN fragments i.  bf16: the lane groups of two
// fragments exchange halves so that a lane stores 8 neighbouring outputs, and a store covers 64 instead of 32 bytes of each row.
template <typename TO, int TN, int TM>
__device__ __forceinline__ void store_rows(const LinearArgs& a, int64_t m, int64_t n, int q, const f32x4 (&acc)[TN][TM], int j) {
    if constexpr (sizeof(TO) == 2 && TN % 2 == 0) {
        if (a.vec == 8 && n + TN * 16 <= a.N) {
#pragma unroll
            for (int i = 0; i < TN; i += 2) {
                uint32_t w[2][2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    f32x4 v = acc[i + h][j];
                    if (a.bias) {
                        const float* b = a.bias + n + (i + h) * 16 + 4 * q;
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] += b[e];
                    }
                    const bf16x4 o = {(bf16)v[0], (bf16)v[1], (bf16)v[2], (bf16)v[3]};
                    const uint2 u = __builtin_bit_cast(uint2, o);
                    w[h][0] = u.x;
                    w[h][1] = u.y;
                }
                // after the swap of odd 16-lane rows of fragment i with even ones of fragment i + 1, group q holds columns
                // (q / 2) * 8 .. +7 of fragment i + q % 2: the first half in [0], the second in [1]
                const auto lo = __builtin_amdgcn_permlane16_swap(w[0][0], w[1][0], false, false), hi = __builtin_amdgcn_permlane16_swap(w[0][1], w[1][1], false, false);
                if (m < a.M)
                    *reinterpret_cast<u32x4*>(static_cast<bf16*>(a.y) + m * a.ldy + n + (i + (q & 1)) * 16 + (q >> 1) * 8) = u32x4{lo[0], hi[0], lo[1], hi[1]};
            }
            return;
        }
    }
#pragma unroll
    for (int i = 0; i < TN; ++i) store_outputs<TO>(a, m, n + i * 16 + 4 * q, acc[i][j]);
}

// Few outputs in all: a workgroup computes 16 outputs of 16 rows, its waves share the slices.  Weights go straight from memory to the matrix
// instruction, AHEAD slices of a wave at a time: lane l holds the 32 values (16 bytes) of row l % 16 in the block l / 16 of the slice.
// FUSED: up to kFusedRows rows of x are packed by every workgroup for itself while its first weights are on their way, which
// saves a launch; the packed rows stay in LDS.  Both in the same call, 8192 x 8192: one row 9.2 against 11.1 us with a launch of its
// own, two 10.4 / 11.1, four 17.7 / 14.9.
// One row is bound by the weights: 8192 x 8192 (35.7 MB) in 9.2 us, 3.9 TB/s; the time beyond the 5 us of the bytes is start, the
// packing's latency and the join of the waves.
constexpr int kFusedRows = 2, kFusedBytes = 32768;

template <typename TO, typename TX, int WAVES, int AHEAD, bool FUSED>
__global__ __launch_bounds__(WAVES * 64) void mxfp4_rows_kernel(const LinearArgs a, const TX* __restrict__ xm, int64_t ldx, int cols) {
    extern __shared__ __align__(16) char lds[];
    __shared__ f32x4 part[WAVES][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * 16, m0 = (int64_t)blockIdx.y * 16;
    const int64_t n = n0 + r < a.N ? n0 + r : a.N - 1, m = m0 + r < a.M ? m0 + r : a.M - 1;
    const uint8_t *wp = a.w + n * a.ldc + q * 16, *xp = a.x + m * a.ldc + q * 16;
    u32x4 wv[AHEAD];
    uint32_t sw[AHEAD];
    auto fetch = [&](int s0) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int s = s0 + u * WAVES < a.slices ? s0 + u * WAVES : a.slices - 1;
            wv[u] = *reinterpret_cast<const u32x4*>(wp + (int64_t)s * 64);
            sw[u] = a.ws[(int64_t)s * a.N + n];
        }
    };
    fetch(wave);
    uint32_t* xc = reinterpret_cast<uint32_t*>(lds);                               // packed rows, then their scales [slice][row]
    uint32_t* xs = xc + (int)a.M * a.slices * 16;
    if constexpr (FUSED) {
        const int per_row = a.slices * 16, items = (int)a.M * per_row;
        for (int item = threadIdx.x; item < items; item += WAVES * 64) {           // groups of 16 lanes stay together
            const int row = item / per_row, i = item - row * per_row;
            uint32_t byte;
            xc[item] = pack_eight<TX>(xm + row * ldx, i * 8, cols, byte);
            const uint32_t b1 = __shfl(byte, (lane & 48) + 4, 64), b2 = __shfl(byte, (lane & 48) + 8, 64), b3 = __shfl(byte, (lane & 48) + 12, 64);
            if ((i & 15) == 0) xs[(i >> 4) * (int)a.M + row] = byte | (b1 << 8) | (b2 << 16) | (b3 << 24);
        }
        __syncthreads();
    }
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = wave; s0 < a.slices; s0 += AHEAD * WAVES) {
        if (s0 != wave) fetch(s0);
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int s = s0 + u * WAVES;
            if (s >= a.slices) break;
            u32x4 xv;
            uint32_t sx;
            if constexpr (FUSED) {
                xv = *reinterpret_cast<const u32x4*>(lds + (int)m * a.slices * 64 + s * 64 + q * 16);
                sx = xs[s * (int)a.M + (int)m];
            } else {
                xv = *reinterpret_cast<const u32x4*>(xp + (int64_t)s * 64);
                sx = a.xs[(int64_t)s * a.xs_rows + m];
            }
            acc = mfma_fp4(wv[u], xv, acc, sw[u] >> (8 * q), sx >> (8 * q));
        }
    }
    part[wave][lane] = acc;
    __syncthreads();
    if (wave == 0) {
        acc = part[0][lane];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) acc += part[w][lane];
        store_outputs<TO>(a, m0 + r, n0 + 4 * q, acc);
    }
}

// Many outputs: a workgroup of WM x WN waves computes BM rows x BN outputs.  Each stage of LDS holds two slices (256 values, 128 bytes
// a row) of both operands and is filled by LDS DMA.  The eight 16-byte blocks of a row lie at block ^ (row % 8), which spreads the 16
// rows of a fragment over all banks; the DMA writes LDS in lane order, so the permutation is applied to its source addresses.
// Scales: LDS [slice of the stage][row] dwords, of which a lane reads the byte of its block.
//
// The loop is skewed: while the products of one slice run, every fragment register is refilled for the next slice as soon as its
// last product has been issued, so the matrix pipe does not wait for LDS.  The one barrier of a stage stands between its two
// slices: the second slice's fragments are in registers by then, so the stage may be overwritten behind it, and the next stage,
// requested STAGES - 1 stages earlier, has landed.  The transfers are spread over the products of the second slice.
template <int BM, int BN> struct TileLds {
    static constexpr int kData = (BM + BN) * 128, kScale = (BM + BN) * 8, kStage = kData + kScale;
};

// 16 (4) bytes per lane from base + off to lds_addr + 16 (4) * lane, invisible to the compiler's dependence tracking: the kernel
// waits for them itself before the barrier that publishes the stage.  lds_addr and base are the same for the whole wave.
// M0 holds the LDS address; nothing else in this kernel uses it.
__device__ __forceinline__ void dma16(const void* base, uint32_t off, uint32_t lds_addr) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds_addr));
}
__device__ __forceinline__ void dma4(const void* base, uint32_t off, uint32_t lds_addr) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" ::"v"(off), "s"(base), "s"(lds_addr));
}

// 256 x 256 tiles by eight waves (128 x 64 outputs each) reach 4.4 PFLOP/s at 8192^3 (250 us); a loop of these matrix instructions
// alone runs at 7.2.  The matrix units are busy 63 % of the time.  Without the transfers the loop is 19 % faster, with half the
// fragment reads 9 %, without the scales 6 %; bank conflicts are 0; the width of the stripes, wave priorities and a 4 x 2 layout of
// the waves change nothing.
// Two waves per SIMD in the launch bounds: with more registers to give away the accumulators went to the other half of the register
// file and were moved about in the loop (128 tile, 8192 -> 8192, 256 rows: 29 -> 26 us).
template <typename TO, int BM, int BN, int WM, int WN, bool WIDE, int STAGES>
__global__ __launch_bounds__(WM * WN * 64, 2) void mxfp4_tile_kernel(const LinearArgs a, int tiles_m, int tiles_n) {
    constexpr int W = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16, kRows = BM + BN;
    constexpr int kStage = TileLds<BM, BN>::kStage, kData = TileLds<BM, BN>::kData;
    // WIDE: the scales of 256 rows of a slice in one transfer (their rows come in fours), else of 64 rows.  With fewer transfers than
    // waves some waves repeat another's: a branch around it would cost more.
    constexpr int kScaleRows = WIDE ? 256 : 64, kScalePieces = kRows * 2 / kScaleRows;
    constexpr int kLoads = kRows / 8 / W, kScaleLoads = (kScalePieces + W - 1) / W, kPieces = kLoads + kScaleLoads;
    static_assert(BM % (8 * W) == 0 && BN % (8 * W) == 0 && BN % 64 == 0 && BM % 64 == 0 && kRows % kScaleRows == 0 && TM >= TN, "whole DMA transfers per wave");
    extern __shared__ __align__(16) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, q = lane >> 4;

    // Workgroups go to the 8 XCDs in turn: each XCD takes one contiguous eighth of the tiles, and walks it in stripes of 8 tiles
    // along n so that the tiles in flight on its 32 CUs share rows of both operands in its L2.
    const int total = tiles_m * tiles_n, per = total / 8, extra = total % 8, xcd = blockIdx.x % 8;
    const int t = xcd * per + (xcd < extra ? xcd : extra) + blockIdx.x / 8;
    const int stripe = t / (8 * tiles_m), within = t - stripe * 8 * tiles_m, width = tiles_n - stripe * 8 < 8 ? tiles_n - stripe * 8 : 8;
    const int64_t m0 = (int64_t)(within / width) * BM, n0 = (int64_t)(stripe * 8 + within % width) * BN;

    // rows of the stage: 0..BN-1 weights, BN..BN+BM-1 inputs (beyond the last row: the last row again, never stored)
    const int block = (lane & 7) ^ (lane >> 3);                 // source block of this lane's slot (rows of a transfer start at multiples of 8)
    // an odd last slice comes as the second of its stage, behind its predecessor, which is not used again; a single slice takes both places
    const int last_slice = a.slices > 1 ? a.slices - 2 : 0, span = a.slices > 1 ? 1 : 0;
    const uint32_t fold = span ? 0 : (block & 4) * 16;
    uint32_t off[kLoads], soff[kScaleLoads];
    const uint32_t* sp[kScaleLoads];        // scales of this wave's transfers in the first slice
    const uint8_t *wp = a.w + n0 * a.ldc, *xp = a.x + m0 * a.ldc;
    const int last_n = (int)(a.N - 1 - n0 < BN ? a.N - 1 - n0 : BN), last_m = (int)(a.M - 1 - m0 < BM ? a.M - 1 - m0 : BM);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {                          // transfer i of this wave: rows (i*W + wave)*8 .. +8
        const int row = (i * W + wave) * 8 + (lane >> 3);
        const int rel = i * W * 8 < BN ? (row < last_n ? row : last_n) : (row - BN < last_m ? row - BN : last_m);
        off[i] = (uint32_t)rel * (uint32_t)a.ldc + block * 16 - fold;
    }
#pragma unroll
    for (int i = 0; i < kScaleLoads; ++i) {                     // kScaleRows rows of one slice
        const int p = (i * W + wave) % kScalePieces, sub = p / (kRows / kScaleRows) * span, row = p % (kRows / kScaleRows) * kScaleRows;
        const bool w = row < BN;
        sp[i] = w ? a.ws + n0 + (int64_t)sub * a.N : a.xs + m0 + (int64_t)sub * a.xs_rows;
        const int64_t left = (w ? a.N - n0 : a.xs_rows - m0) - kScaleRows / 64;
        const int rel = (w ? row : row - BN) + lane * (kScaleRows / 64);
        soff[i] = (uint32_t)(rel < left ? rel : (int)left) * 4;
    }
    const uint32_t lds0 = (uint32_t)(size_t)(const __attribute__((address_space(3))) char*)lds;
    // piece i of this wave for the stage of slices 2 step and 2 step + 1
    auto fill = [&](int step, int i) {
        const int slice = 2 * step < last_slice ? 2 * step : last_slice;
        const uint32_t at = lds0 + step % STAGES * kStage;
        if (i < kLoads) {
            dma16((i * W * 8 < BN ? wp : xp) + slice * 64, off[i < kLoads ? i : 0], at + (i * W + wave) * 1024);
        } else {
            const int e = i < kLoads ? 0 : i - kLoads, p = (e * W + wave) % kScalePieces;
            const int64_t rows = p % (kRows / kScaleRows) * kScaleRows < BN ? a.N : a.xs_rows;
            if constexpr (WIDE) dma16(sp[e] + slice * rows, soff[e], at + kData + p * kScaleRows * 4);
            else dma4(sp[e] + slice * rows, soff[e], at + kData + p * kScaleRows * 4);
        }
    };

    f32x4 acc[TN][TM];
    const int nw = (wave % WN) * TN * 16, mw = BN + (wave / WN) * TM * 16;      // this wave's first fragment rows
    const int steps = (a.slices + 1) / 2;
    u32x4 fw[2][TN], fx[TM];
    uint32_t sw[2][TN], sx[TM];
    // All but the youngest `pending` stages of this wave have landed and its reads are done; behind the barrier this holds for all waves
    auto publish = [&](auto pending) {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(pending() * kPieces) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    // The products of the fragments in set h; meanwhile the other set is refilled from slice `half` of stage `next`, and stage
    // `ahead` is requested.
    auto multiply = [&](auto h, int next, int half, auto request, int ahead) {
        // fragment rows are r modulo 16, so r modulo 8 decides the slot
        const char* d = lds + next % STAGES * kStage + r * 128 + ((half * 4 + q) ^ (r & 7)) * 16;
        const char* c = lds + next % STAGES * kStage + kData + half * kRows * 4 + r * 4 + q;
#pragma unroll
        for (int j = 0; j < TM; ++j) {
#pragma unroll
            for (int i = 0; i < TN; ++i) acc[i][j] = mfma_fp4(fw[h()][i], fx[j], acc[i][j], sw[h()][i], sx[j]);
            __builtin_amdgcn_sched_barrier(0);
            fx[j] = *reinterpret_cast<const u32x4*>(d + (mw + j * 16) * 128);
            sx[j] = *reinterpret_cast<const uint8_t*>(c + (mw + j * 16) * 4);
            if (j < TN) {
                fw[1 - h()][j] = *reinterpret_cast<const u32x4*>(d + (nw + j * 16) * 128);
                sw[1 - h()][j] = *reinterpret_cast<const uint8_t*>(c + (nw + j * 16) * 4);
            }
            if constexpr (request()) {
#pragma unroll
                for (int i = j * kPieces / TM; i < (j + 1) * kPieces / TM; ++i) fill(ahead, i);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    constexpr std::integral_constant<int, 0> first{};
    constexpr std::integral_constant<int, 1> second{};
    const bool odd = a.slices & 1;
    constexpr std::integral_constant<int, 0> none{};
    for (int s = 0; s < STAGES && s < steps; ++s) {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) fill(s, i);
    }
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (steps >= STAGES) publish(std::integral_constant<int, STAGES - 1>{});
    else publish(none);
    {
        const char* d = lds + r * 128 + (q ^ (r & 7)) * 16;
        const char* c = lds + kData + r * 4 + q;
#pragma unroll
        for (int j = 0; j < TM; ++j) {
            fx[j] = *reinterpret_cast<const u32x4*>(d + (mw + j * 16) * 128);
            sx[j] = *reinterpret_cast<const uint8_t*>(c + (mw + j * 16) * 4);
        }
#pragma unroll
        for (int i = 0; i < TN; ++i) {
            fw[0][i] = *reinterpret_cast<const u32x4*>(d + (nw + i * 16) * 128);
            sw[0][i] = *reinterpret_cast<const uint8_t*>(c + (nw + i * 16) * 4);
        }
    }
    int step = 0;
    for (; step + STAGES < steps; ++step) {
        multiply(first, step, 1, std::false_type{}, 0);
        publish(std::integral_constant<int, STAGES - 2>{});
        multiply(second, step + 1, step + 2 == steps && odd ? 1 : 0, std::true_type{}, step + STAGES);
    }
    for (; step < steps; ++step) {       // the last stages; what is read ahead of the end is not used
        multiply(first, step, 1, std::false_type{}, 0);
        if (step + 1 == steps && odd) break;
        publish(none);
        multiply(second, step + 1, step + 2 == steps && odd ? 1 : 0, std::false_type{}, 0);
    }
    const int64_t m = m0 + (wave / WN) * TM * 16 + r, n = n0 + (wave % WN) * TN * 16;
#pragma unroll
    for (int j = 0; j < TM; ++j) store_rows<TO, TN, TM>(a, m + j * 16, n, q, acc, j);
}

// ------------------------------------------------------------------------------------------------ host
static int64_t slices_of(int64_t cols) { return (cols + kSlice - 1) / kSlice; }

// The kernel for M rows and N outputs: 16 = the rows kernel, else the side of the square tile.
// Rows kernel: while its workgroups of 16 x 16 outputs are few (two per CU), splitting the slices over 8 or 16 waves beats a tile that
// walks them alone; beyond, the weights are read again for every 16 rows, or too many short-lived workgroups fetch them.  Rows kernel /
// 64-tile, us, packed x: 8192 -> 512: 64 rows 6.3/11.5, 256 rows (512 workgroups) 10.5/11.7; 8192 -> 2048: 64 (512) 10.4/11.7, 100
// (896) 17.5/11.9; 8192 -> 8192: 16 (512) 10.8/12.0, 33 (1536) 24.5/12.1; 2048 -> 131072, one row (8192): 39/23; 1664 -> 1000: 33 rows
// 3.6/4.8, 128 rows (504) 5.0/4.9; 512 -> 2048: 64 rows (512) 4.0/3.8.
// Tiles: a larger one moves fewer bytes per product, if it does not leave CUs without work and its rows are not mostly empty.  64 /
// 128 / 256, us: 8192 -> 32768: 64 rows 24/29/46, 128 rows (256 tiles of 128) 32/31/46, 1000 rows (512 tiles of 256) 224/155/121;
// 8192 -> 8192: 256 rows (128 tiles of 128) 19/26/44, 1000 rows (512 of 128, 128 of 256) 61/41/50.
static int kernel_of(int64_t M, int64_t N) {
    if (((M + 15) / 16) * ((N + 15) / 16) <= 512) return 16;
    for (int t : {256, 128}) {
        if (M > t / 2 && ((M + t - 1) / t) * ((N + t - 1) / t) >= 256) return t;
    }
    return 64;
}
static bool packs_inside(int64_t M, int64_t K, int64_t N) { return M <= kFusedRows && M * slices_of(K) * 68 <= kFusedBytes && kernel_of(M, N) == 16; }

static int check_matrix(const char* who, int dtype, const void* x, int64_t ld, int64_t rows, int64_t cols) {
    SEGK_REQUIRE(x, SEGK_EINVAL, "%s: null pointer", who);
    SEGK_REQUIRE(dtype == SEGK_F32 || dtype == SEGK_BF16, SEGK_EINVAL, "%s: unknown dtype %d", who, dtype);
    SEGK_REQUIRE(rows > 0 && cols > 0 && rows < (1ll << 31) && cols < (1ll << 30), SEGK_ESHAPE, "%s: bad shape", who);
    SEGK_REQUIRE(ld >= cols, SEGK_ESHAPE, "%s: ld smaller than a row", who);
    SEGK_REQUIRE(reinterpret_cast<uintptr_t>(x) % esize(dtype) == 0, SEGK_EALIGN, "%s: matrix is not aligned to its type", who);
    return SEGK_OK;
}
static int check_packed(const char* who, const void* codes, const void* scales) {
    SEGK_REQUIRE(codes && scales, SEGK_EINVAL, "%s: null pointer", who);
    SEGK_REQUIRE(aligned16(codes), SEGK_EALIGN, "%s: codes must be 16-byte aligned", who);
    SEGK_REQUIRE(reinterpret_cast<uintptr_t>(scales) % 4 == 0, SEGK_EALIGN, "%s: scales must be 4-byte aligned", who);
    return SEGK_OK;
}

// f(first row, rows) for pieces of at most 2^31 - 1 items
template <typename F> static int by_rows(int64_t rows, int64_t per_row, F&& f) {
    const int64_t most = ((1ll << 31) - 256) / per_row;
    for (int64_t r0 = 0; r0 < rows; r0 += most) {
        if (const int rc = f(r0, rows - r0 < most ? rows - r0 : most)) return rc;
    }
    return SEGK_OK;
}

static int quantize(int dtype, const void* x, int64_t ld, int64_t rows, int64_t cols, void* codes, void* scales, int64_t scale_rows, hipStream_t st) {
    const int64_t per_row = slices_of(cols) * 16;
    return by_rows(rows, per_row, [&](int64_t r0, int64_t n) -> int {
        const uint32_t items = (uint32_t)(n * per_row);
        SEGK_DISPATCH_DTYPE(dtype, T, hipLaunchKernelGGL((mxfp4_quantize_kernel<T>), dim3((items + 255) / 256), dim3(256), 0, st, (const T*)x, ld,
                                                         (int)cols, items, Divide((uint32_t)per_row), scale_rows, r0, (uint32_t*)codes, (uint32_t*)scales));
        SEGK_LAUNCH_CHECK();
        return SEGK_OK;
    });
}

template <typename TO, int BM, int BN, int WM, int WN, bool WIDE, int STAGES> static int launch_tile(const LinearArgs& a, hipStream_t st) {
    constexpr int bytes = STAGES * TileLds<BM, BN>::kStage;
    const int64_t tm = (a.M + BM - 1) / BM, tn = (a.N + BN - 1) / BN;
    auto kernel = mxfp4_tile_kernel<TO, BM, BN, WM, WN, WIDE, STAGES>;
    if constexpr (bytes > 65536) {
        static std::atomic<bool> allowed[64] = {};               // once per device
        int dev = 0;
        SEGK_HIP(hipGetDevice(&dev));
        if (dev >= 64 || !allowed[dev].load(std::memory_order_acquire)) {
            SEGK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
            if (dev < 64) allowed[dev].store(true, std::memory_order_release);
        }
    }
    hipLaunchKernelGGL(kernel, dim3((unsigned)(tm * tn)), dim3(WM * WN * 64), bytes, st, a, (int)tm, (int)tn);
    SEGK_LAUNCH_CHECK();
    return SEGK_OK;
}


}  // namespace segk

using namespace segk;

extern "C" size_t segk_mxfp4_codes_bytes(int64_t rows, int64_t cols) { return rows > 0 && cols > 0 ? (size_t)(rows * slices_of(cols) * 64) : 0; }
extern "C" size_t segk_mxfp4_scales_bytes(int64_t rows, int64_t cols) { return rows > 0 && cols > 0 ? (size_t)(rows * slices_of(cols) * 4) : 0; }

extern "C" int segk_mxfp4_quantize(int dtype, const void* x, int64_t ld, int64_t rows, int64_t cols, void* codes, void* scales, int dev, void* stream) {
    if (const int rc = check_matrix("mxfp4_quantize", dtype, x, ld, rows, cols)) return rc;
    if (const int rc = check_packed("mxfp4_quantize", codes, scales)) return rc;
    SEGK_USE_DEVICE(dev);
    return quantize(dtype, x, ld, rows, cols, codes, scales, rows, (hipStream_t)stream);
}

extern "C" int segk_mxfp4_dequantize(int dtype, const void* codes, const void* scales, int64_t rows, int64_t cols, void* y, int64_t ld, int dev,
                                     void* stream) {
    if (const int rc = check_matrix("mxfp4_dequantize", dtype, y, ld, rows, cols)) return rc;
    if (const int rc = check_packed("mxfp4_dequantize", codes, scales)) return rc;
    SEGK_USE_DEVICE(dev);
    const int64_t per_row = slices_of(cols) * 16;
    return by_rows(rows, per_row, [&](int64_t r0, int64_t n) -> int {
        const uint32_t items = (uint32_t)(n * per_row);
        SEGK_DISPATCH_DTYPE(dtype, T, hipLaunchKernelGGL((mxfp4_dequantize_kernel<T>), dim3((items + 255) / 256), dim3(256), 0, (hipStream_t)stream,
                                                         (const uint32_t*)codes, (const uint8_t*)scales, (int)cols, items,
                                                         Divide((uint32_t)per_row), rows, r0, (T*)y, ld));
        SEGK_LAUNCH_CHECK();
        return SEGK_OK;
    });
}

extern "C" size_t segk_mxfp4_linear_workspace(int64_t M, int64_t K, int64_t N) {
    if (packs_inside(M, K, N)) return 0;
    return align_up(segk_mxfp4_codes_bytes(M, K), 16) + segk_mxfp4_scales_bytes((int64_t)align_up(M > 0 ? M : 0, 4), K);
}

extern "C" int segk_mxfp4_linear(const void* x, int x_dtype, int64_t ldx, const void* x_codes, const void* x_scales, int64_t M, int64_t K,
                                 const void* w_codes, const void* w_scales, int64_t N, const float* bias, void* y, int y_dtype, int64_t ldy,
                                 void* workspace, size_t workspace_bytes, int dev, void* stream) {
    SEGK_REQUIRE((x != nullptr) != (x_codes != nullptr), SEGK_EINVAL, "mxfp4_linear: either x or x_codes is given");
    SEGK_REQUIRE(M > 0 && K > 0 && N > 0 && M < (1ll << 28) && N < (1ll << 28) && K < (1ll << 24), SEGK_ESHAPE, "mxfp4_linear: bad shape");
    if (const int rc = check_matrix("mxfp4_linear", y_dtype, y, ldy, M, N)) return rc;
    if (const int rc = check_packed("mxfp4_linear", w_codes, w_scales)) return rc;
    if (x) {
        if (const int rc = check_matrix("mxfp4_linear", x_dtype, x, ldx, M, K)) return rc;
        SEGK_REQUIRE(packs_inside(M, K, N) || (workspace && workspace_bytes >= segk_mxfp4_linear_workspace(M, K, N)), SEGK_EWORKSPACE, "mxfp4_linear: workspace too small");
        SEGK_REQUIRE(aligned16(workspace), SEGK_EALIGN, "mxfp4_linear: workspace must be 16-byte aligned");
    } else if (const int rc = check_packed("mxfp4_linear", x_codes, x_scales)) return rc;
    const int choice = kernel_of(M, N);
    // a launch has fewer than 2^32 threads; those of the rows kernel are few
    SEGK_REQUIRE(choice == 16 || ((M + choice - 1) / choice) * ((N + choice - 1) / choice) < (1ll << 32) / (choice == 256 ? 512 : 256), SEGK_ESHAPE,
                 "mxfp4_linear: too many outputs for one launch");
    SEGK_USE_DEVICE(dev);
    hipStream_t st = (hipStream_t)stream;
    const bool pack_inside = x && packs_inside(M, K, N);
    if (x && !pack_inside) {
        x_codes = workspace;
        x_scales = (const uint8_t*)workspace + align_up(segk_mxfp4_codes_bytes(M, K), 16);
        if (const int rc = quantize(x_dtype, x, ldx, M, K, workspace, const_cast<void*>(x_scales), (int64_t)align_up(M, 4), st)) return rc;
    }
    LinearArgs a = {};
    a.w = (const uint8_t*)w_codes; a.ws = (const uint32_t*)w_scales; a.x = (const uint8_t*)x_codes; a.xs = (const uint32_t*)x_scales;
    a.bias = bias; a.y = y; a.M = M; a.N = N; a.xs_rows = x && !pack_inside ? (int64_t)align_up(M, 4) : M; a.ldc = slices_of(K) * 64; a.ldy = ldy; a.slices = (int)slices_of(K);
    for (int v : {4, 8})
        if (reinterpret_cast<uintptr_t>(y) % (v * esize(y_dtype)) == 0 && ldy % v == 0) a.vec = v;
    const bool wide = N % 4 == 0 && a.xs_rows % 4 == 0 && aligned16(w_scales) && aligned16(x_scales);
    SEGK_DISPATCH_DTYPE(y_dtype, TO, {
        if (choice == 256 && wide) return launch_tile<TO, 256, 256, 2, 4, true, 2>(a, st);
        if (choice == 256) return launch_tile<TO, 256, 256, 2, 4, false, 2>(a, st);
        if (choice == 128) return launch_tile<TO, 128, 128, 2, 2, false, 2>(a, st);
        // Up to two tiles per CU wait for memory rather than for each other: four stages instead of the room for four workgroups per
        // CU.  2 / 4 stages, us: 8192 -> 8192, 64 rows (128 tiles) 18.9/12.2, 256 rows (512) 21.0/18.8, 1000 rows (2048) 61/67.
        if (choice == 64 && ((M + 63) / 64) * ((N + 63) / 64) <= 512) return launch_tile<TO, 64, 64, 2, 2, false, 4>(a, st);
        if (choice == 64) return launch_tile<TO, 64, 64, 2, 2, false, 2>(a, st);
        const dim3 grid((unsigned)((N + 15) / 16), (unsigned)((M + 15) / 16));
        // Up to 4096 outputs there are few workgroups, and 16 waves share the slices of each; beyond, 8 waves, with 8 slices in flight
        // if they are many.  One row of packed x, 8192 outputs from 8192 values: (8 waves, 8 ahead) 8.8, (8, 4) 9.6, (4, 8) 12.2,
        // (16, 8) 13.5 us; from 512 values: (8, 4) 3.3, (8, 8) 4.1 us; 512 outputs from 8192: (16, 4) 4.7, (16, 8) 6.6 us.
        auto launch = [&](auto waves, auto ahead) {
            if (pack_inside) {
                const unsigned bytes = (unsigned)(M * a.slices * 68);
                if (x_dtype == SEGK_BF16)
                    hipLaunchKernelGGL((mxfp4_rows_kernel<TO, bf16, waves(), ahead(), true>), grid, dim3(waves() * 64), bytes, st, a, (const bf16*)x, ldx, (int)K);
                else
                    hipLaunchKernelGGL((mxfp4_rows_kernel<TO, float, waves(), ahead(), true>), grid, dim3(waves() * 64), bytes, st, a, (const float*)x, ldx, (int)K);
            } else {
                hipLaunchKernelGGL((mxfp4_rows_kernel<TO, float, waves(), ahead(), false>), grid, dim3(waves() * 64), 0, st, a, (const float*)nullptr, (int64_t)0, 0);
            }
        };
        if (N <= 4096) launch(std::integral_constant<int, 16>{}, std::integral_constant<int, 4>{});
        else if (a.slices > 32) launch(std::integral_constant<int, 8>{}, std::integral_constant<int, 8>{});
        else launch(std::integral_constant<int, 8>{}, std::integral_constant<int, 4>{});
    });
    SEGK_LAUNCH_CHECK();
    return SEGK_OK;
}
