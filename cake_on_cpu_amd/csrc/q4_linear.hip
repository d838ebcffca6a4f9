// q4_linear.hip -- y[M][N] = x[M][K] . v[N][K]^T (+ bias) with v in 4 bits (packed form: q4_kernels.hip)
// for a few rows of x, and the choice between this and the kernel for many (q4_linear_bands.hip).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "kernels.hpp"
#include "q4_operands.hpp"

namespace cake {

namespace {

// The scales (or zero points) of one row and block as they lie, fetched ahead and read where they are used
template <int GPB, bool WIDE>
struct GroupValues {
    static constexpr int WORDS = WIDE ? GPB : (GPB + 1) / 2;
    struct alignas(WIDE ? 4 * GPB : 2 * GPB) Packed { unsigned char bytes[WIDE ? 4 * GPB : 2 * GPB]; };
    unsigned w[WORDS];
    __device__ __forceinline__ void load(const unsigned char* base, unsigned row)
    {
        const Packed p = reinterpret_cast<const Packed*>(base)[row];
        if constexpr (sizeof(Packed) >= 4) __builtin_memcpy(w, &p, sizeof(Packed));
        else w[0] = __builtin_bit_cast(unsigned short, p);
    }
    __device__ __forceinline__ float at(int g, bool half) const
    {
        if (WIDE) return __builtin_bit_cast(float, w[g]);
        const unsigned narrow = w[g >> 1] >> ((g & 1) * 16) & 0xFFFFu;
        return half ? (float)__builtin_bit_cast(_Float16, (unsigned short)narrow) : __builtin_bit_cast(float, narrow << 16);
    }
};

struct StreamArgs {
    const void* x;
    const unsigned char* q;
    const void* bias;
    void* y;
    Q4Layout lay;
    int M, with_zeros;
    int chunk_blocks;     // blocks of 128 columns of x held in LDS at a time, a multiple of the waves
    int zero_at;          // byte offset in LDS of 16 zero bytes, behind the chunk
    bool vec;
};

// Few rows of x (up to 16 of pieces): the codes are read once, straight into the registers of the wave that
// multiplies them, x lies in LDS as the matrix pipe's A operand.  A workgroup owns NT tiles of 16
// rows of v; its waves share the blocks of 128 columns out among them in turn, DEPTH turns in
// flight each, and add their sums up through LDS in a fixed order.
// Row r of pieces is A's row 4 (r & 3) + (r >> 2), so that the first four rows come out in the four lanes'
// first result register and REGS registers cover 4 REGS rows: with one token the scale costs two
// operations per group instead of eight.
template <int TYPE, int GPB, bool WIDE, int REGS, int NT>
__global__ __launch_bounds__(1024) void linear_q4_stream_kernel(StreamArgs a)
{
    typedef typename Element<TYPE>::T T;
    constexpr int PIECES = pieces_of<TYPE>();
    constexpr int SG = 4 / GPB;
    constexpr int DEPTH = 4 / NT;
    extern __shared__ __align__(16) unsigned char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int quad = lane >> 4, col = lane & 15;
    const int K = a.lay.K, blocks = a.lay.blocks;
    const int rows = a.M * PIECES;
    const int tile0 = blockIdx.x * NT;

    // this lane's row of the A operand, or the zeros
    const int my_row = (col & 3) * 4 + (col >> 2);
    const unsigned a_base = my_row < rows ? my_row * 64 + quad * 16 : a.zero_at;
    const unsigned a_step = my_row < rows ? rows * 64 : 0;
    if (threadIdx.x < 4) reinterpret_cast<unsigned*>(lds + a.zero_at)[threadIdx.x] = 0;

    struct Held {
        uintx4 code[NT];
        GroupValues<GPB, WIDE> s[NT], z[NT];
    } held[DEPTH];
    // addresses are scalars that move on by the waves' number of blocks, and a lane's place in a block
    constexpr int SCALE_BYTES = 16 * GPB * (WIDE ? 4 : 2);
    const bool half = a.lay.scale_type == CAKE_HIP_F16;
    const unsigned char *code_at[NT], *scale_at[NT], *zero_at[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const size_t unit = (size_t)min(tile0 + nt, a.lay.tiles - 1) * blocks + wave;
        code_at[nt] = a.q + unit * 1024;
        scale_at[nt] = a.q + a.lay.scales_at + unit * SCALE_BYTES;
        zero_at[nt] = a.q + a.lay.zeros_at + unit * SCALE_BYTES;
    }
    int fetched = wave;
    auto fetch = [&](Held& h) {
        if (fetched < blocks) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                h.code[nt] = __builtin_nontemporal_load(reinterpret_cast<const uintx4*>(code_at[nt] + (unsigned)lane * 16));
                h.s[nt].load(scale_at[nt], col);
                if (a.with_zeros) h.z[nt].load(zero_at[nt], col);
                code_at[nt] += waves * 1024;
                scale_at[nt] += waves * SCALE_BYTES;
                zero_at[nt] += waves * SCALE_BYTES;
            }
        }
        fetched += waves;
    };

    floatx4 acc[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) acc[nt] = floatx4{0, 0, 0, 0};
    uintx4 ones;
#pragma unroll
    for (int i = 0; i < 4; ++i) ones[i] = Codes<TYPE>::ONES;

    auto multiply = [&](const Held& h, int step0) {
#pragma unroll
        for (int g = 0; g < GPB; ++g) {
            floatx4 p[NT], sum = floatx4{0, 0, 0, 0};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) p[nt] = floatx4{0, 0, 0, 0};
#pragma unroll
            for (int i = g * SG; i < (g + 1) * SG; ++i) {
                const uintx4 xa = *reinterpret_cast<const uintx4*>(lds + a_base + a_step * (unsigned)(step0 + i));
                sum = Codes<TYPE>::mfma(xa, ones, sum);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) p[nt] = Codes<TYPE>::mfma(xa, unpack_codes<TYPE>(h.code[nt][i]), p[nt]);
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const float s = h.s[nt].at(g, half), z = a.with_zeros ? h.z[nt].at(g, half) : 8.f;
#pragma unroll
                for (int r = 0; r < REGS; ++r) acc[nt][r] = __builtin_fmaf(s, __builtin_fmaf(-z, sum[r], p[nt][r]), acc[nt][r]);
            }
        }
    };

    const int turns = (blocks + waves - 1) / waves, turns_per_chunk = a.chunk_blocks / waves;
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) fetch(held[d]);
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
                    for (int m = 0; m < a.M; ++m)
                        for (int part = threadIdx.x; part < parts; part += blockDim.x) {
                            const int k = chunk0 * 128 + part * 8;
                            T v[8];
                            load_eight<TYPE>(static_cast<const T*>(a.x) + (size_t)m * K + k, K - k, a.vec, v);
#pragma unroll
                            for (int p = 0; p < PIECES; ++p)
                                *reinterpret_cast<uintx4*>(lds + ((part >> 2) * rows + m * PIECES + p) * 64 + (part & 3) * 16) = piece_of<TYPE>(v, p);
                        }
                    __syncthreads();
                }
                --until_chunk;
                if (block < blocks) multiply(held[d], (block - chunk0) * 4);
                fetch(held[d]);
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
        for (int r = 0; r < REGS; ++r) {
            const int row = r * 4 + quad;
            if (row < rows) red[(wave * rows + row) * WIDTH + nt * 16 + col] = acc[nt][r];
        }
    __syncthreads();
    for (int i = threadIdx.x; i < a.M * WIDTH; i += blockDim.x) {
        const int m = i / WIDTH, c = i - m * WIDTH, n = tile0 * 16 + c;
        if (n >= a.lay.N) continue;
        float v = 0;
        for (int w = 0; w < waves; ++w)
#pragma unroll
            for (int p = 0; p < PIECES; ++p) v += red[(w * rows + m * PIECES + p) * WIDTH + c];
        if (a.bias) v += (float)static_cast<const T*>(a.bias)[n];
        static_cast<T*>(a.y)[(size_t)m * a.lay.N + n] = (T)v;
    }
}

template <int TYPE, int GPB>
hipError_t stream_launch(StreamArgs a, hipStream_t stream)
{
    const int rows = a.M * pieces_of<TYPE>();
    // two tiles a workgroup share x and its column sums, as soon as that leaves a workgroup for every compute unit
    const int nt = a.lay.tiles >= 512 ? 2 : 1;
    int waves = nt == 1 ? 16 : 8;
    while (waves > 1 && waves / 2 >= a.lay.blocks) waves /= 2;
    // a chunk of x of at most 32 KB (one turn of the waves at least)
    const int block_bytes = rows * 256;
    const int all_turns = (a.lay.blocks + waves - 1) / waves;
    const int turns = std::max(1, std::min(all_turns, 32 * 1024 / (block_bytes * waves)));
    a.chunk_blocks = turns * waves;
    a.zero_at = a.chunk_blocks * block_bytes;
    const size_t lds = std::max((size_t)waves * rows * nt * 16 * 4, (size_t)a.zero_at + 16);
    const dim3 grid((a.lay.tiles + nt - 1) / nt), block(64 * waves);
    auto run = [&](auto kernel) {
        if (lds > 64 * 1024) {
            hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
            if (e != hipSuccess) return e;
        }
        kernel<<<grid, block, lds, stream>>>(a);
        return hipGetLastError();
    };
    auto of_width = [&](auto wide) {
        constexpr bool W = decltype(wide)::value;
        if (rows <= 4) return nt == 1 ? run(&linear_q4_stream_kernel<TYPE, GPB, W, 1, 1>) : run(&linear_q4_stream_kernel<TYPE, GPB, W, 1, 2>);
        return nt == 1 ? run(&linear_q4_stream_kernel<TYPE, GPB, W, 4, 1>) : run(&linear_q4_stream_kernel<TYPE, GPB, W, 4, 2>);
    };
    return a.lay.scale_type == CAKE_HIP_F32 ? of_width(std::true_type()) : of_width(std::false_type());
}

// One tile of 16 rows of pieces is streamed; K == 0 is only a bias, which the streaming kernel writes for any M
bool streams(int M, int K, int type) { return K == 0 || M <= (type == CAKE_HIP_F32 ? 5 : 16); }

}  // namespace

size_t linear_q4_workspace(int M, int N, int K, int type)
{
    return M == 0 || N == 0 || streams(M, K, type) ? 0 : linear_q4_bands_workspace(M, N, K, type);
}

hipError_t launch_linear_q4(const void* x, const void* q, const void* bias, void* y, int type, int M, const Q4Layout& lay,
                            bool with_zeros, void* workspace, hipStream_t stream)
{
    const bool vec = lay.K % 8 == 0 && (uintptr_t)x % 16 == 0;
    hipError_t e = hipSuccess;
    if (streams(M, lay.K, type)) {
        StreamArgs a{};
        a.x = x;
        a.q = static_cast<const unsigned char*>(q);
        a.bias = bias;
        a.y = y;
        a.lay = lay;
        a.M = M;
        a.with_zeros = with_zeros;
        a.vec = vec;
        q4_for_type_and_group(type, lay.groups_per_block,
                              [&](auto t, auto gpb) { e = stream_launch<decltype(t)::value, decltype(gpb)::value>(a, stream); });
        return e;
    }
    return launch_linear_q4_bands(x, q, bias, y, type, M, lay, with_zeros, workspace, vec, stream);
}

}  // namespace cake
