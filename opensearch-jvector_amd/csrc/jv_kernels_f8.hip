// jv_kernels_f8.hip — rows of 8-bit floats with one scale for each block of 128 components: encode, decode, and the product of a batch of
// queries with such rows (gfx950).
//
// A block of x is held as e4m3 codes c and one exponent byte b:  x ~ c 2^(b - 127),  2^(b - 127) the least power of two with
// max|x| <= 448 * 2^(b - 127)  (448: the largest e4m3 value).  A power of two, because the matrix instruction takes such a scale as an
// operand and because it makes both directions exact but for the one rounding to e4m3.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "jv_mm.h"
#include "jv_mm_out.h"

using namespace jvmm;

// ---------------------------------------------------------------------------------------------
// A half-wave holds one block, four components a lane: the block's maximum is five exchanges, a store is 4 B of codes.  A workgroup's eight
// half-waves take `rounds` runs of eight blocks: sixteen in long calls, one where there are few blocks.  Loads and stores need no alignment.
// 1 000 003 x 1 000 float32: 1.12 ms, 4.5 TB/s (a large copy: 4.7); back: 0.99 ms, 5.1 TB/s.
// ---------------------------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ f32x4 load4(const T* row, int at, int d) {
    f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
    if (at + 3 < d) {
        if constexpr (sizeof(T) == 4) {
            __builtin_memcpy(&x, row + at, 16);
        } else {
            bf16x4 v;
            __builtin_memcpy(&v, row + at, 8);
#pragma unroll
            for (int e = 0; e < 4; e++) x[e] = (float)v[e];
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (at + e < d) x[e] = (float)row[at + e];
    }
    return x;
}

template <typename T>
__global__ __launch_bounds__(256) void jvf_encode_kernel(const T* __restrict__ x, int64_t stride, int64_t blocks, int d, int nb, int rounds,
                                                         uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    const int hw = threadIdx.x >> 5, l = threadIdx.x & 31;
    const int64_t first = (int64_t)blockIdx.x * (rounds * 8);
    const int64_t row0 = first / nb;
    const uint32_t b0 = (uint32_t)(first - row0 * nb);
    for (int i = 0; i < rounds; i++) {
        const int64_t blk = first + i * 8 + hw;
        if (blk >= blocks) break;   // (whole half-waves: the exchanges below stay inside one)
        const uint32_t at = b0 + (uint32_t)(i * 8 + hw), up = at / (uint32_t)nb, b = at - up * (uint32_t)nb;
        const f32x4 v = load4(x + (row0 + up) * stride, (int)b * 128 + l * 4, d);
        // the largest finite magnitude, compared as bits
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const uint32_t bits = __float_as_uint(v[e]) & 0x7fffffffu;
            top = bits < 0x7f800000u && bits > top ? bits : top;
        }
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) {
            const uint32_t other = (uint32_t)__shfl_xor((int)top, off, 64);
            top = other > top ? other : top;
        }
        // top = 1.m 2^(e - 127): 2^(e - 135) reaches 1.75 2^8 = 448, the next one the rest (a subnormal maximum ends at byte 0)
        int byte = (int)(top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
        byte = byte < 0 ? 0 : byte;
        byte = top == 0 ? 127 : byte;
        const float inv = __uint_as_float((uint32_t)(254 - byte) << 23);
        int c = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inv, v[1] * inv, 0, false);
        c = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inv, v[3] * inv, c, true);
        uint32_t code = (uint32_t)c;
#pragma unroll
        for (int e = 0; e < 4; e++)   // e4m3 has no infinity: what is not finite becomes its NaN
            if ((__float_as_uint(v[e]) & 0x7f800000u) == 0x7f800000u) code = (code & ~(0xffu << (8 * e))) | (0x7fu << (8 * e));
        *(uint32_t*)(codes + blk * 128 + l * 4) = code;
        if (l == 0) scales[blk] = (uint8_t)byte;
    }
}

template <typename T>
__global__ __launch_bounds__(256) void jvf_decode_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int64_t blocks,
                                                         int d, int nb, int rounds, T* __restrict__ x, int64_t stride) {
    const int hw = threadIdx.x >> 5, l = threadIdx.x & 31;
    const int64_t first = (int64_t)blockIdx.x * (rounds * 8);
    const int64_t row0 = first / nb;
    const uint32_t b0 = (uint32_t)(first - row0 * nb);
    for (int i = 0; i < rounds; i++) {
        const int64_t blk = first + i * 8 + hw;
        if (blk >= blocks) break;
        const uint32_t p = b0 + (uint32_t)(i * 8 + hw), up = p / (uint32_t)nb, b = p - up * (uint32_t)nb;
        const int code = *(const int*)(codes + blk * 128 + l * 4);
        const uint32_t byte = scales[blk];
        const float s = byte == 0 ? __uint_as_float(0x00400000u) : byte == 255 ? __uint_as_float(0x7fc00000u) : __uint_as_float(byte << 23);
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(code, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(code, true);
        const f32x4 v = {lo[0] * s, lo[1] * s, hi[0] * s, hi[1] * s};
        const int at = (int)b * 128 + l * 4;
        T* out = x + (row0 + up) * stride + at;
        if (at + 3 < d) {
            if constexpr (sizeof(T) == 4) {
                __builtin_memcpy(out, &v, 16);
            } else {
                const bf16x4 h = {(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
                __builtin_memcpy(out, &h, 8);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (at + e < d) out[e] = (T)v[e];
        }
    }
}

// runs of eight blocks for each workgroup: eight workgroups a CU before a workgroup gets more than one
static int rounds_of(int64_t blocks) { return (int)std::min<int64_t>(std::max<int64_t>(blocks / (8 * 2048), 1), 16); }

extern "C" hipError_t jvk_f8_encode(const void* x, int dtype, int64_t stride, int64_t n, int d, uint8_t* codes, uint8_t* scales, hipStream_t s) {
    const int nb = (d + 127) / 128;
    const int64_t blocks = n * nb;
    const int rounds = rounds_of(blocks);
    const int64_t grid = (blocks + rounds * 8 - 1) / (rounds * 8);
    if (grid <= 0) return hipSuccess;
    if (grid > 0x7fffffffll) return hipErrorInvalidValue;
    if (dtype == 0) jvf_encode_kernel<float><<<(unsigned)grid, 256, 0, s>>>((const float*)x, stride, blocks, d, nb, rounds, codes, scales);
    else jvf_encode_kernel<__bf16><<<(unsigned)grid, 256, 0, s>>>((const __bf16*)x, stride, blocks, d, nb, rounds, codes, scales);
    return hipGetLastError();
}

extern "C" hipError_t jvk_f8_decode(const uint8_t* codes, const uint8_t* scales, int64_t n, int d, void* x, int dtype, int64_t stride, hipStream_t s) {
    const int nb = (d + 127) / 128;
    const int64_t blocks = n * nb;
    const int rounds = rounds_of(blocks);
    const int64_t grid = (blocks + rounds * 8 - 1) / (rounds * 8);
    if (grid <= 0) return hipSuccess;
    if (grid > 0x7fffffffll) return hipErrorInvalidValue;
    if (dtype == 0) jvf_decode_kernel<float><<<(unsigned)grid, 256, 0, s>>>(codes, scales, blocks, d, nb, rounds, (float*)x, stride);
    else jvf_decode_kernel<__bf16><<<(unsigned)grid, 256, 0, s>>>(codes, scales, blocks, d, nb, rounds, (__bf16*)x, stride);
    return hipGetLastError();
}

// bf16 scores keep 8 bits: the 8-bit unit's sums are enough.  float32 scores take the bf16 unit (jv_mm.h).  Tiles: 256 x 256 where they fill the
// chip, more than half of one is queries and the output's rows are 16-B aligned (jv_pipe.h); 32 x 128 and 64 x 128 for up to 32 and 64 queries (the
// rows are streamed); 128 x 128 otherwise, but 64 x 64 where that is no more than one tile a CU.
//   1 x 100 000 x 768: 22 us, the launches of the two calls (the query's encoding and this) and 77 MB of codes.
//   256 x 500 000 x 768, float32: 265 us, 3.4 TB/s, more than half of it the scores; the stores of one tile and the products of the next
//     share a wave's order of memory operations, so they overlap by two phases only.  d = 128: 133 us, 4.3 TB/s (large copy: 4.7).
//   4096 x 65 536 x 1536, bf16: 470 us, 1750 TFLOP/s (a large library product of 8-bit floats: 2785).  The matrix unit has work in 42 % of the cycles; 15 %
//     of the LDS cycles are bank conflicts (float32 scores: 25 %), which bf16 products on these tiles do not have: the scales' reads or the
//     epilogue's writes, not found out which.  256 x 256 against 128 x 128 tiles: 1024 x 100 000 x 768, bf16: 128 and 178 us.
template <int TY>
static hipError_t score(const JvMmOut& a, hipStream_t s) {
    const int64_t M = a.mm.M, N = a.mm.N, tiles = (M + 127) / 128 * ((N + 127) / 128);
    if (M > 128 && (M + 255) / 256 * ((N + 255) / 256) >= 192 && N >= 16 && aligned_rows(a)) return mm_out_pipe<TY>(a, s);
    if (M <= 32) return tiles <= 256 ? mm_out_tile<Tile<TY, 1, 1, 1, 4, 4>>(a, s) : mm_out_tile<Tile<TY, 1, 1, 1, 4, 2>>(a, s);
    if (tiles <= 256) return mm_out_tile<Tile<TY, 1, 1, 2, 2, 4>>(a, s);
    return M <= 64 ? mm_out_tile<Tile<TY, 2, 1, 1, 4, 2>>(a, s) : mm_out_tile<Tile<TY, 2, 2, 2, 2, 2>>(a, s);
}
extern "C" hipError_t jvk_f8_score(const JvMmOut* a, hipStream_t s) { return a->dtype == 0 ? score<F8W>(*a, s) : score<F8>(*a, s); }
