// q4_linear.hip -- y[M][N] = x[M][K] . v[N][K]^T (+ bias) with v in 4 bits (packed form: q4_kernels.hip).
//
// Codes are whole numbers 0..15, exact in 16-bit floats, so the products go to the matrix pipe as
// x . code and the group's scale and zero point are applied to the 32-bit sums behind it:
//   y[m][n] = sum over groups g of s[n][g] * (sum_k x[m][k] code[n][k] - z[n][g] * sum_k x[m][k]).
// The second inner sum is one more matrix product, with a column of ones: it lands in the lane that
// needs it.  No weight is rounded.  x is exact as well: 16-bit types go in as they are, a 32-bit x
// as three bf16 pieces (its leading, middle and last 8 significant bits, cut, not rounded, so that
// no piece overflows) that take three rows of the product and are added up at the end.
#include <hip/hip_runtime.h>

#include "kernels.hpp"
#include "low_bits.hpp"

namespace cake {

namespace {

template <int TYPE> struct Codes;   // what the matrix pipe multiplies
template <> struct Codes<CAKE_HIP_F16> {
    typedef f16x8 V;
    static __device__ __forceinline__ unsigned pair(unsigned bytes, bool upper)
    {
        return upper ? __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(bytes, 512.f, true))
                     : __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(bytes, 512.f, false));
    }
    static constexpr unsigned ONES = 0x3C003C00u;
    static __device__ __forceinline__ floatx4 mfma(uintx4 a, uintx4 b, floatx4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b), c, 0, 0, 0);
    }
};
template <> struct Codes<CAKE_HIP_BF16> {
    typedef bf16x8 V;
    static __device__ __forceinline__ unsigned pair(unsigned bytes, bool upper)
    {
        return upper ? __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(bytes, 512.f, true))
                     : __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(bytes, 512.f, false));
    }
    static constexpr unsigned ONES = 0x3F803F80u;
    static __device__ __forceinline__ floatx4 mfma(uintx4 a, uintx4 b, floatx4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b), c, 0, 0, 0);
    }
};
template <> struct Codes<CAKE_HIP_F32> : Codes<CAKE_HIP_BF16> {};

template <int TYPE> constexpr int pieces_of() { return TYPE == CAKE_HIP_F32 ? 3 : 1; }

template <int TYPE>
__device__ __forceinline__ uintx4 unpack_codes(unsigned word)
{
    const unsigned low = word & 0x0F0F0F0Fu, high = (word >> 4) & 0x0F0F0F0Fu;
    uintx4 b;
    b[0] = Codes<TYPE>::pair(low, false);
    b[1] = Codes<TYPE>::pair(low, true);
    b[2] = Codes<TYPE>::pair(high, false);
    b[3] = Codes<TYPE>::pair(high, true);
    return b;
}

// eight consecutive elements of a row of x, zero from column K on
template <int TYPE>
__device__ __forceinline__ void load_eight(const typename Element<TYPE>::T* at, int left, bool vec, typename Element<TYPE>::T (&v)[8])
{
    typedef typename Element<TYPE>::T T;
    if (vec && left >= 8) {
        struct alignas(16) Eight { T e[8]; } got = *reinterpret_cast<const Eight*>(at);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = got.e[e];
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < left ? at[e] : (T)0.f;
    }
}

// piece p of eight elements as the matrix pipe takes them
template <int TYPE>
__device__ __forceinline__ uintx4 piece_of(const typename Element<TYPE>::T (&v)[8], int p)
{
    uintx4 out;
    if constexpr (TYPE == CAKE_HIP_F32) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            unsigned half[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float rest = v[e + j];
                unsigned cut = __builtin_bit_cast(unsigned, rest) & 0xFFFF0000u;
                for (int i = 0; i < p; ++i) {
                    rest -= __builtin_bit_cast(float, cut);   // exact: the bits behind the cut
                    cut = __builtin_bit_cast(unsigned, rest) & 0xFFFF0000u;
                }
                half[j] = cut;
            }
            out[e / 2] = (half[0] >> 16) | half[1];
        }
    } else {
        struct alignas(16) Eight { typename Element<TYPE>::T e[8]; } all;
#pragma unroll
        for (int e = 0; e < 8; ++e) all.e[e] = v[e];
        out = __builtin_bit_cast(uintx4, all);
    }
    return out;
}

template <int GPB> struct GroupPair { float s[GPB], z[GPB]; };

template <int GPB>
__device__ __forceinline__ void load_groups(const void* base, size_t at, int type, float (&out)[GPB])
{
    if (type == CAKE_HIP_F32) {
        struct alignas(4 * GPB) P { float v[GPB]; } p = reinterpret_cast<const P*>(base)[at];
#pragma unroll
        for (int g = 0; g < GPB; ++g) out[g] = p.v[g];
    } else {
        struct alignas(2 * GPB) P { unsigned short v[GPB]; } p = reinterpret_cast<const P*>(base)[at];
#pragma unroll
        for (int g = 0; g < GPB; ++g)
            out[g] = type == CAKE_HIP_F16 ? (float)__builtin_bit_cast(_Float16, p.v[g]) : __builtin_bit_cast(float, (unsigned)p.v[g] << 16);
    }
}

struct StreamArgs {
    const void* x;
    const unsigned char* q;
    const void* bias;
    void* y;
    Q4Layout lay;
    int M, with_zeros;
    int tokens;           // rows of x of one workgroup
    int bands;            // workgroups along x's rows; those of one strip of weights run together
    int chunk_blocks;     // blocks of 128 columns of x held in LDS at a time, a multiple of the waves
    int zero_at;          // byte offset in LDS of 16 zero bytes, behind the chunk
    bool vec;
};

// Few rows of x: the codes are read once, straight into the registers of the wave that multiplies
// them, x lies in LDS as the matrix pipe's A operand.  A workgroup owns NT tiles of 16 rows of v
// and up to 16 MT rows (of pieces) of x; its waves share the blocks of 128 columns out among them in
// turn, four blocks in flight each, and add their sums up through LDS in a fixed order.
// Row r of pieces is A's row 4 (r & 3) + (r >> 2), so that the first four rows come out in the four lanes'
// first result register and REGS registers cover 4 REGS rows: with one token the scale costs two
// operations per group instead of eight.
template <int TYPE, int GPB, int MT, int REGS, int NT>
__global__ __launch_bounds__(512) void linear_q4_stream_kernel(StreamArgs a)
{
    typedef typename Element<TYPE>::T T;
    constexpr int PIECES = pieces_of<TYPE>();
    constexpr int SG = 4 / GPB;
    constexpr int DEPTH = NT == 1 ? 4 : 2;
    extern __shared__ __align__(16) unsigned char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int quad = lane >> 4, col = lane & 15;
    const int K = a.lay.K, blocks = a.lay.blocks;
    const int strip = (int)(blockIdx.x / (unsigned)a.bands), band = (int)(blockIdx.x - (unsigned)strip * (unsigned)a.bands);
    const int m0 = band * a.tokens;
    const int tokens = min(a.tokens, a.M - m0);
    const int rows = tokens * PIECES;
    const int tile0 = strip * NT;

    // this lane's row of the A operand in each tile of 16, or the zeros
    unsigned a_base[MT], a_step[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const int r = mt * 16 + (col & 3) * 4 + (col >> 2);
        a_base[mt] = r < rows ? r * 64 + quad * 16 : a.zero_at;
        a_step[mt] = r < rows ? rows * 64 : 0;
    }
    if (threadIdx.x < 4) reinterpret_cast<unsigned*>(lds + a.zero_at)[threadIdx.x] = 0;

    struct Held {
        uintx4 code[NT];
        float s[NT][GPB], z[NT][GPB];
    } held[DEPTH];
    auto fetch = [&](Held& h, int block) {
        if (block >= blocks) return;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int tile = min(tile0 + nt, a.lay.tiles - 1);
            const size_t unit = (size_t)tile * blocks + block;
            h.code[nt] = __builtin_nontemporal_load(reinterpret_cast<const uintx4*>(a.q + unit * 1024 + lane * 16));
            load_groups<GPB>(a.q + a.lay.scales_at, unit * 16 + col, a.lay.scale_type, h.s[nt]);
            if (a.with_zeros) load_groups<GPB>(a.q + a.lay.zeros_at, unit * 16 + col, a.lay.scale_type, h.z[nt]);
        }
    };

    floatx4 acc[NT][MT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) acc[nt][mt] = floatx4{0, 0, 0, 0};
    uintx4 ones;
#pragma unroll
    for (int i = 0; i < 4; ++i) ones[i] = Codes<TYPE>::ONES;

    auto multiply = [&](const Held& h, int step0) {
#pragma unroll
        for (int g = 0; g < GPB; ++g) {
            floatx4 p[NT][MT], sum[MT];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                sum[mt] = floatx4{0, 0, 0, 0};
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) p[nt][mt] = floatx4{0, 0, 0, 0};
            }
#pragma unroll
            for (int i = g * SG; i < (g + 1) * SG; ++i) {
                uintx4 b[NT];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) b[nt] = unpack_codes<TYPE>(h.code[nt][i]);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    const uintx4 xa = *reinterpret_cast<const uintx4*>(lds + a_base[mt] + a_step[mt] * (unsigned)(step0 + i));
                    sum[mt] = Codes<TYPE>::mfma(xa, ones, sum[mt]);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) p[nt][mt] = Codes<TYPE>::mfma(xa, b[nt], p[nt][mt]);
                }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const float s = h.s[nt][g], z = a.with_zeros ? h.z[nt][g] : 8.f;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int r = 0; r < REGS; ++r)
                        acc[nt][mt][r] = __builtin_fmaf(s, __builtin_fmaf(-z, sum[mt][r], p[nt][mt][r]), acc[nt][mt][r]);
            }
        }
    };

    const int turns = (blocks + waves - 1) / waves, turns_per_chunk = a.chunk_blocks / waves;
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) fetch(held[d], wave + d * waves);
    int block = wave, chunk0 = 0, until_chunk = 0;
    for (int t0 = 0; t0 < turns; t0 += DEPTH) {
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            if (t0 + d < turns) {   // the same for every wave of the workgroup
                if (until_chunk == 0) {
                    chunk0 = (t0 + d) * waves;
                    until_chunk = turns_per_chunk;
                    if (chunk0) __syncthreads();
                    // the next chunk of x: piece p of row m at [step of 32 columns][m * PIECES + p][8-column part]
                    const int parts = min(a.chunk_blocks, blocks - chunk0) * 16;
                    for (int i = threadIdx.x; i < tokens * parts; i += blockDim.x) {
                        const int m = i / parts, part = i - m * parts;
                        const int k = chunk0 * 128 + part * 8;
                        T v[8];
                        load_eight<TYPE>(static_cast<const T*>(a.x) + (size_t)(m0 + m) * K + k, K - k, a.vec, v);
#pragma unroll
                        for (int p = 0; p < PIECES; ++p)
                            *reinterpret_cast<uintx4*>(lds + ((part >> 2) * rows + m * PIECES + p) * 64 + (part & 3) * 16) = piece_of<TYPE>(v, p);
                    }
                    __syncthreads();
                }
                --until_chunk;
                if (block < blocks) multiply(held[d], (block - chunk0) * 4);
                fetch(held[d], block + DEPTH * waves);
                block += waves;
            }
        }
    }

    // the waves' sums side by side in LDS, then one thread per result: waves and pieces in order
    __syncthreads();
    float* red = reinterpret_cast<float*>(lds);
    constexpr int WIDTH = NT * 16;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int r = 0; r < REGS; ++r) {
                const int row = mt * 16 + r * 4 + quad;
                if (row < rows) red[(wave * rows + row) * WIDTH + nt * 16 + col] = acc[nt][mt][r];
            }
    __syncthreads();
    for (int i = threadIdx.x; i < tokens * WIDTH; i += blockDim.x) {
        const int m = i / WIDTH, c = i - m * WIDTH, n = tile0 * 16 + c;
        if (n >= a.lay.N) continue;
        float v = 0;
        for (int w = 0; w < waves; ++w)
#pragma unroll
            for (int p = 0; p < PIECES; ++p) v += red[(w * rows + m * PIECES + p) * WIDTH + c];
        if (a.bias) v += (float)static_cast<const T*>(a.bias)[n];
        static_cast<T*>(a.y)[(size_t)(m0 + m) * a.lay.N + n] = (T)v;
    }
}

template <int TYPE, int GPB>
hipError_t stream_launch(StreamArgs a, int cus, hipStream_t stream)
{
    constexpr int PIECES = pieces_of<TYPE>();
    const int rows = a.M * PIECES;
    const int mt = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
    const int nt = mt == 1 ? 1 : 2;
    a.tokens = a.M < mt * 16 / PIECES ? a.M : mt * 16 / PIECES;
    const int wg_rows = a.tokens * PIECES;
    const int strips = (a.lay.tiles + nt - 1) / nt, bands = (int)(((long long)a.M + a.tokens - 1) / a.tokens);
    a.bands = bands;
    int waves = mt == 4 ? 4 : 8;
    while (waves > 1 && waves / 2 >= a.lay.blocks) waves /= 2;
    // a chunk of x of at most 32 KB (one turn of the waves at least)
    const int block_bytes = wg_rows * 256;
    int turns = (32 * 1024) / (block_bytes * waves);
    if (turns < 1) turns = 1;
    const int all_turns = (a.lay.blocks + waves - 1) / waves;
    if (turns > all_turns) turns = all_turns;
    a.chunk_blocks = turns * waves;
    a.zero_at = a.chunk_blocks * block_bytes;
    const size_t red_bytes = (size_t)waves * wg_rows * nt * 16 * 4;
    const size_t lds = red_bytes > (size_t)a.zero_at + 16 ? red_bytes : (size_t)a.zero_at + 16;
    const dim3 grid((unsigned)strips * (unsigned)bands), block(64 * waves);
    auto run = [&](auto kernel) {
        if (lds > 64 * 1024) {
            hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
            if (e != hipSuccess) return e;
        }
        kernel<<<grid, block, lds, stream>>>(a);
        return hipGetLastError();
    };
    if (rows <= 4) return run(&linear_q4_stream_kernel<TYPE, GPB, 1, 1, 1>);
    if (mt == 1) return run(&linear_q4_stream_kernel<TYPE, GPB, 1, 4, 1>);
    if (mt == 2) return run(&linear_q4_stream_kernel<TYPE, GPB, 2, 4, 2>);
    return run(&linear_q4_stream_kernel<TYPE, GPB, 4, 4, 2>);
}

}  // namespace

size_t linear_q4_workspace(int M, int N, int K, int type)
{
    (void)M, (void)N, (void)K, (void)type;
    return 0;
}

hipError_t launch_linear_q4(const void* x, const void* q, const void* bias, void* y, int type, int M, const Q4Layout& lay,
                            bool with_zeros, void* workspace, int cus, hipStream_t stream)
{
    (void)workspace;
    StreamArgs a{};
    a.x = x;
    a.q = static_cast<const unsigned char*>(q);
    a.bias = bias;
    a.y = y;
    a.lay = lay;
    a.M = M;
    a.with_zeros = with_zeros;
    a.vec = lay.K % 8 == 0 && (uintptr_t)x % 16 == 0;
    hipError_t e = hipSuccess;
    q4_for_type_and_group(type, lay.groups_per_block,
                          [&](auto t, auto gpb) { e = stream_launch<decltype(t)::value, decltype(gpb)::value>(a, cus, stream); });
    return e;
}

}  // namespace cake
