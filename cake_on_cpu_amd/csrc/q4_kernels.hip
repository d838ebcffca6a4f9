// q4_kernels.hip -- weights of a linear layer in 4 bits: quantising, packing, unpacking.
//
// Value of code c in 0..15 at row n, column k: v = (c - z) * s with the scale s and the zero point
// z of the row's run of `group` columns k / group (z = 8 where none are kept).
//
// Packed form.  Rows are taken 16 at a time (a tile), columns 128 at a time (a block); a block of a
// tile is 1 KB, blocks of a tile follow one another, and so do tiles.  Lane l of a wave owns 16
// bytes of a block at l * 16: row l & 15, and in its dword i the eight columns 32 i + 8 (l >> 4) + e,
// e = 0..7.  That is the B operand of v_mfma_f32_16x16x32 for step i, so a wave fetches four steps
// of a tile with one coalesced 16-byte load a lane and every step lies in one group of 32 columns or
// more.  Inside a dword, byte b has element b in its low and element b + 4 in its high nibble:
// a mask (and a shift) leaves four codes as four bytes, and a byte 0..15 read as an 8-bit float
// (4 exponent and 3 mantissa bits, bias 7) is code * 2^-9 exactly -- 0..7 as subnormals, 8..15 with
// the exponent's last bit -- so the hardware's conversion of two such bytes with a scale of 2^9 gives
// two codes as 16-bit floats (or in units of 2^-12, with 2^-3): 7 vector instructions for 8 weights.
// Behind the codes (at the next multiple of 256 bytes) lie the scales as [tile][block][row][128 / group]
// in their own type, then the zero points likewise.  Rows past N and columns past K hold code 0
// under scale 0.
#include <hip/hip_runtime.h>

#include "kernels.hpp"
#include "low_bits.hpp"

namespace cake {

namespace {

// element e of a dword sits at this bit
__device__ __forceinline__ int nibble_at(int e) { return e < 4 ? 8 * e : 8 * (e - 4) + 4; }

// round(w / s), ties to even, of the real quotient.  r is within one of it; w - r s is exact in one
// fused operation for |r| < 32 (a multiple of the smaller last place of the two, and below 2^24
// of those), so comparing it with half of s decides without a division.
__device__ __forceinline__ float round_quotient(float w, float s, float inv)
{
    float r = __builtin_rintf(w * inv);
    const float rest = 2.f * __builtin_fmaf(-r, s, w);
    const bool odd = ((int)r & 1) != 0;
    if (rest > s || (rest == s && odd)) r += 1.f;
    else if (rest < -s || (rest == -s && odd)) r -= 1.f;
    return r;
}

// a / by for a constant `by`: the product with the rounded reciprocal is within one last place, and one
// correction by the exact remainder makes it the correctly rounded quotient (Markstein's theorem);
// 3 operations where a division in 64 bits takes about thirty.
__device__ __forceinline__ double quotient(double a, double by)
{
    const double y = 1.0 / by, q = a * y;
    return __builtin_fma(__builtin_fma(-by, q, a), y, q);
}

__device__ __forceinline__ float larger_or_nan(float a, float b) { return (b > a || b != b) ? b : a; }

__device__ __forceinline__ float as_kept(float v, int type)
{
    if (type == CAKE_HIP_F16) return (float)(_Float16)v;
    if (type == CAKE_HIP_BF16) return (float)(__bf16)v;
    return v;
}

// One wave per block of 16 rows x 128 columns, each lane its 4 x 8 columns of one row: the four
// lanes of a row are 16 apart, so a group's extremes are two shuffles away.  Bound by memory: reads
// w once (128 contiguous bytes of a row per step), writes half a byte a weight.
template <int TYPE, int GPB>
__global__ __launch_bounds__(256) void q4_quantize_kernel(const typename Element<TYPE>::T* __restrict__ w, unsigned char* __restrict__ q,
                                                          Q4Layout lay, int with_zeros)
{
    typedef typename Element<TYPE>::T T;
    const int lane = threadIdx.x & 63;
    const size_t unit = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (unit >= (size_t)lay.tiles * lay.blocks) return;
    const int tile = (int)(unit / lay.blocks), block = (int)(unit - (size_t)tile * lay.blocks);
    const int row = tile * 16 + (lane & 15), quad = lane >> 4;
    float v[4][8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int k = block * 128 + 32 * i + 8 * quad;
        const T* at = w + (size_t)row * lay.K + k;
        if (row < lay.N && k + 8 <= lay.K) {
            T got[8];
            __builtin_memcpy(got, at, sizeof got);   // 16-byte loads, which the hardware takes at any address
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] = (float)got[e];
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] = row < lay.N && k + e < lay.K ? (float)at[e] : 0.f;
        }
    }
    constexpr int SG = 4 / GPB;   // steps of 32 columns in a group
    uintx4 codes;
    float keep_s[GPB], keep_z[GPB];
#pragma unroll
    for (int g = 0; g < GPB; ++g) {
        float hi = 0.f, lo = 0.f;
#pragma unroll
        for (int i = g * SG; i < (g + 1) * SG; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                hi = larger_or_nan(hi, v[i][e]);
                lo = larger_or_nan(lo, -v[i][e]);
            }
#pragma unroll
        for (int step = 16; step <= 32; step *= 2) {
            hi = larger_or_nan(hi, __shfl_xor(hi, step));
            lo = larger_or_nan(lo, __shfl_xor(lo, step));
        }
        // range / 15 and maximum / 7, each rounded once to 32 bits, then to the type the scale is kept in
        float s = with_zeros ? (float)quotient((double)hi + (double)lo, 15.0) : (float)quotient((double)larger_or_nan(hi, lo), 7.0);
        s = as_kept(s, lay.scale_type);
        // a scale so small that its reciprocal overflows: both sides of the quotient times 2^64, exactly
        const float up = s < 1e-30f ? 18446744073709551616.f : 1.f;
        const float su = s * up, inv = 1.f / su;
        const float z = !with_zeros ? 8.f : s > 0.f ? __builtin_fminf(__builtin_fmaxf(round_quotient(lo * up, su, inv), 0.f), 15.f) : 8.f;
#pragma unroll
        for (int i = g * SG; i < (g + 1) * SG; ++i) {
            unsigned word = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float r = s > 0.f ? round_quotient(v[i][e] * up, su, inv) : 0.f;
                const float c = __builtin_fminf(__builtin_fmaxf(r + z, 0.f), 15.f);
                word |= (unsigned)(int)c << nibble_at(e);
            }
            codes[i] = word;
        }
        const bool real = row < lay.N && (block * GPB + g) * (128 / GPB) < lay.K;
        if (!real) {   // nothing of the matrix: code 0 under scale 0
#pragma unroll
            for (int i = g * SG; i < (g + 1) * SG; ++i) codes[i] = 0;
        }
        keep_s[g] = real ? s : 0.f;
        keep_z[g] = real ? z : 0.f;
    }
    *reinterpret_cast<uintx4*>(q + unit * 1024 + lane * 16) = codes;
    if (quad == 0) {
#pragma unroll
        for (int g = 0; g < GPB; ++g) {
            const size_t at = (unit * 16 + lane) * GPB + g;
            store_from_float(q + lay.scales_at, at, lay.scale_type, keep_s[g]);
            if (with_zeros) store_from_float(q + lay.zeros_at, at, lay.scale_type, keep_z[g]);
        }
    }
}

// w[n][k] = (code - z) * s.  The difference of a code and a zero point that is a whole number is exact; the
// product is rounded to 32 bits and then to w's type.
template <int TYPE, int GPB>
__global__ __launch_bounds__(256) void q4_dequantize_kernel(const unsigned char* __restrict__ q, typename Element<TYPE>::T* __restrict__ w,
                                                            Q4Layout lay, int with_zeros)
{
    typedef typename Element<TYPE>::T T;
    const int lane = threadIdx.x & 63;
    const size_t unit = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (unit >= (size_t)lay.tiles * lay.blocks) return;
    const int tile = (int)(unit / lay.blocks), block = (int)(unit - (size_t)tile * lay.blocks);
    const int row = tile * 16 + (lane & 15), quad = lane >> 4;
    const uintx4 codes = *reinterpret_cast<const uintx4*>(q + unit * 1024 + lane * 16);
    if (row >= lay.N) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int k = block * 128 + 32 * i + 8 * quad;
        const size_t at = (unit * 16 + (lane & 15)) * GPB + i * GPB / 4;
        const float s = load_as_float(q + lay.scales_at, at, lay.scale_type);
        const float z = with_zeros ? load_as_float(q + lay.zeros_at, at, lay.scale_type) : 8.f;
        T out[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float v = ((float)((codes[i] >> nibble_at(e)) & 15u) - z) * s;
            // fp16: the compiler would take product and conversion as one instruction, which rounds
            // once; the value is the product in 32 bits, whatever type it is read as
            if (TYPE == CAKE_HIP_F16) asm("" : "+v"(v));
            out[e] = (T)v;
        }
        T* to = w + (size_t)row * lay.K + k;
        if (k + 8 <= lay.K) {
            __builtin_memcpy(to, out, sizeof out);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (k + e < lay.K) to[e] = out[e];
        }
    }
}

// Eight columns of a checkpoint's row (byte j: column 2 j low, 2 j + 1 high) as a dword of the packed form
__device__ __forceinline__ unsigned reorder_nibbles(unsigned w)
{
    const unsigned even = w & 0x0F0F0F0Fu, odd = w >> 4 & 0x0F0F0F0Fu;   // columns 0 2 4 6 and 1 3 5 7, a byte each
    const unsigned low = (even & 0x00FFu) | (odd & 0x00FFu) << 8 | (even & 0xFF00u) << 8 | (odd & 0xFF00u) << 16;   // 0 1 2 3
    const unsigned high = (even >> 16 & 0x00FFu) | (odd >> 16 & 0x00FFu) << 8 | (even >> 16 & 0xFF00u) << 8 | (odd >> 16 & 0xFF00u) << 16;
    return low | high << 4;
}

// codes[N][(K + 1) / 2] (byte j of a row: column 2 j in the low nibble, 2 j + 1 in the high one), scales and
// zero points [N][groups] into the packed form.  A lane fetches 32 columns of its row, 16 bytes at any
// address, so that the four lanes of a row read 64 bytes in a row; what it keeps is its eight of
// each of the four steps, a 4 x 4 transposition among them.
template <int GPB>
__global__ __launch_bounds__(256) void q4_pack_kernel(const unsigned char* __restrict__ codes, const void* __restrict__ scales,
                                                      const void* __restrict__ zeros, unsigned char* __restrict__ q, Q4Layout lay)
{
    const int lane = threadIdx.x & 63;
    const size_t unit = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (unit >= (size_t)lay.tiles * lay.blocks) return;
    const int tile = (int)(unit / lay.blocks), block = (int)(unit - (size_t)tile * lay.blocks);
    const int row = tile * 16 + (lane & 15), quad = lane >> 4;
    const int k0 = block * 128 + 32 * quad;
    unsigned w[4] = {0, 0, 0, 0};
    if (row < lay.N) {
        const unsigned char* from = codes + (size_t)row * ((lay.K + 1) / 2) + k0 / 2;
        if (k0 + 32 <= lay.K) {
            __builtin_memcpy(w, from, 16);
        } else {
            for (int k = k0; k < lay.K; ++k) {   // (a last column in a byte of its own leaves the byte's other half out)
                const unsigned code = (from[(k - k0) >> 1] >> (4 * (k & 1))) & 15u;
                const int at = k - k0;
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] |= at >> 3 == j ? code << (4 * (at & 7)) : 0u;
            }
        }
    }
    // w[j] of quarter i is columns 32 i + 8 j; wanted in quarter j's w[i]
    auto swap = [&](unsigned& a, unsigned& b, int across) {
        const bool upper = (lane & across) != 0;
        const unsigned got = __shfl_xor(upper ? a : b, across);
        a = upper ? got : a;
        b = upper ? b : got;
    };
    swap(w[0], w[1], 16);
    swap(w[2], w[3], 16);
    swap(w[0], w[2], 32);
    swap(w[1], w[3], 32);
    uintx4 out;
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = reorder_nibbles(w[i]);
    *reinterpret_cast<uintx4*>(q + unit * 1024 + lane * 16) = out;
    if (lane < 16 * GPB) {   // a lane per scale, in the order they are kept
        const int groups = (lay.K + 128 / GPB - 1) / (128 / GPB), n = tile * 16 + lane / GPB, gk = block * GPB + lane % GPB;
        const bool real = n < lay.N && gk < groups;
        const size_t at = unit * 16 * GPB + lane, in = (size_t)n * groups + gk;
        store_from_float(q + lay.scales_at, at, lay.scale_type, real ? load_as_float(scales, in, lay.scale_type) : 0.f);
        if (zeros) store_from_float(q + lay.zeros_at, at, lay.scale_type, real ? load_as_float(zeros, in, lay.scale_type) : 0.f);
    }
}

unsigned q4_grid(const Q4Layout& lay) { return (unsigned)(((size_t)lay.tiles * lay.blocks + 3) / 4); }

}  // namespace

Q4Layout q4_layout(int N, int K, int group, int scale_type, bool with_zeros)
{
    Q4Layout lay;
    lay.N = N;
    lay.K = K;
    lay.tiles = (int)(((long long)N + 15) / 16);
    lay.blocks = (int)(((long long)K + 127) / 128);
    lay.groups_per_block = 128 / group;
    lay.scale_type = scale_type;
    const size_t units = (size_t)lay.tiles * lay.blocks;
    const size_t scale_bytes = (units * 16 * lay.groups_per_block * type_bytes(scale_type) + 255) & ~(size_t)255;
    lay.scales_at = units * 1024;
    lay.zeros_at = lay.scales_at + scale_bytes;
    lay.bytes = lay.zeros_at + (with_zeros ? scale_bytes : 0);
    return lay;
}

hipError_t launch_q4_quantize(const void* w, int w_type, void* q, const Q4Layout& lay, bool with_zeros, hipStream_t stream)
{
    const dim3 grid(q4_grid(lay)), block(256);
    unsigned char* to = static_cast<unsigned char*>(q);
    auto go = [&](auto type, auto gpb) {
        typedef typename Element<decltype(type)::value>::T T;
        q4_quantize_kernel<decltype(type)::value, decltype(gpb)::value><<<grid, block, 0, stream>>>(static_cast<const T*>(w), to, lay, with_zeros);
    };
    q4_for_type_and_group(w_type, lay.groups_per_block, go);
    return hipGetLastError();
}

hipError_t launch_q4_dequantize(const void* q, void* w, int w_type, const Q4Layout& lay, bool with_zeros, hipStream_t stream)
{
    const dim3 grid(q4_grid(lay)), block(256);
    const unsigned char* from = static_cast<const unsigned char*>(q);
    auto go = [&](auto type, auto gpb) {
        typedef typename Element<decltype(type)::value>::T T;
        q4_dequantize_kernel<decltype(type)::value, decltype(gpb)::value><<<grid, block, 0, stream>>>(from, static_cast<T*>(w), lay, with_zeros);
    };
    q4_for_type_and_group(w_type, lay.groups_per_block, go);
    return hipGetLastError();
}

hipError_t launch_q4_pack(const unsigned char* codes, const void* scales, const void* zeros, void* q, const Q4Layout& lay, hipStream_t stream)
{
    const dim3 grid(q4_grid(lay)), block(256);
    auto go = [&](auto, auto gpb) {
        q4_pack_kernel<decltype(gpb)::value><<<grid, block, 0, stream>>>(codes, scales, zeros, static_cast<unsigned char*>(q), lay);
    };
    q4_for_type_and_group(CAKE_HIP_F32, lay.groups_per_block, go);
    return hipGetLastError();
}

}  // namespace cake
