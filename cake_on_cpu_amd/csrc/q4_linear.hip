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
};

// x of one block of 128 columns on its way to the matrix pipe's A operand.  16-bit x: every lane fetches
// its 8 columns of its row for each of the four steps, straight in operand order.  32-bit x: the wave
// fetches two columns a lane, cuts them into pieces and passes them through LDS of its own; no
// other wave takes part, so nothing waits at a barrier.
template <int TYPE, int REGS, int MT>
struct BlockOfX {
    typedef typename Element<TYPE>::T T;
    uintx4 step[MT][4];
    __device__ __forceinline__ void fetch(const T* x, int M, int K, int block, int lane, int my_row)
    {
        const int k = block * 128 + (lane >> 4) * 8;
        const bool whole = block * 128 + 128 <= K;   // the same for the whole wave
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
            for (int i = 0; i < 4; ++i) step[mt][i] = uintx4{0, 0, 0, 0};
            if (my_row + 16 * mt < M) {
                const T* at = x + (size_t)(my_row + 16 * mt) * K + k;
                if (whole) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) __builtin_memcpy(&step[mt][i], at + 32 * i, 16);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        T v[8];
                        load_eight<TYPE>(at + 32 * i, K - k - 32 * i, v);
                        step[mt][i] = piece_of<TYPE>(v, 0);
                    }
                }
            }
        }
    }
    static constexpr int TOKENS = 0;
    __device__ __forceinline__ void to_lds(unsigned char*, int) const {}
    __device__ __forceinline__ uintx4 operand(int mt, int i, const unsigned char*, bool) const { return step[mt][i]; }
};
template <int REGS, int MT>
struct BlockOfX<CAKE_HIP_F32, REGS, MT> {
    static constexpr int TOKENS = REGS == 1 ? 1 : 5 * MT;   // whose pieces fill 4, 16 or 32 rows
    float v[TOKENS][2];
    __device__ __forceinline__ void fetch(const float* x, int M, int K, int block, int lane, int)
    {
        const int k = block * 128 + lane * 2;
        const bool whole = block * 128 + 128 <= K;
#pragma unroll
        for (int m = 0; m < TOKENS; ++m) {
            const float* at = x + (size_t)(m < M ? m : 0) * K + k;
            if (whole) {
                __builtin_memcpy(v[m], at, 8);
            } else {
                v[m][0] = k < K ? at[0] : 0.f;
                v[m][1] = k + 1 < K ? at[1] : 0.f;
            }
        }
    }
    __device__ __forceinline__ void to_lds(unsigned char* mine, int lane) const
    {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // the last block has been read
#pragma unroll
        for (int m = 0; m < TOKENS; ++m) {
            float rest[2] = {v[m][0], v[m][1]};
#pragma unroll
            for (int p = 0; p < 3; ++p) {
                unsigned cut[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    cut[j] = __builtin_bit_cast(unsigned, rest[j]) & 0xFFFF0000u;
                    rest[j] -= __builtin_bit_cast(float, cut[j]);   // exact
                }
                *reinterpret_cast<unsigned*>(mine + ((lane >> 4) * TOKENS * 3 + m * 3 + p) * 64 + (lane & 15) * 4) = cut[0] >> 16 | cut[1];
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    __device__ __forceinline__ uintx4 operand(int mt, int i, const unsigned char* mine_row, bool real) const
    {
        const uintx4 got = *reinterpret_cast<const uintx4*>(mine_row + (real ? mt * 1024 : 0) + i * TOKENS * 3 * 64);
        return real ? got : uintx4{0, 0, 0, 0};
    }
};

// Few rows of x (up to 16 MT of pieces): the codes are read once, straight into the registers of the
// wave that multiplies them.  A workgroup owns NT tiles of 16 rows of v; its waves share the blocks of
// 128 columns out among them in turn, DEPTH turns in flight each, and add their sums up through LDS
// in a fixed order.
// Row r of pieces is A's row 4 (r & 3) + (r >> 2), so that the first four rows come out in the four lanes'
// first result register and REGS registers cover 4 REGS rows: with one token the scale costs two
// operations per group instead of eight.
template <int TYPE, int GPB, bool WIDE, int REGS, int NT, int MT>
__global__ __launch_bounds__(NT * MT == 1 ? 1024 : 512) void linear_q4_stream_kernel(StreamArgs a)
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

    // this lane's row of the A operand, and the place of its columns in the wave's own LDS (32-bit x)
    const int my_row = (col & 3) * 4 + (col >> 2);
    constexpr int OWN = BlockOfX<TYPE, REGS, MT>::TOKENS * 3 * 256;
    unsigned char* mine = lds + wave * OWN;
    const unsigned char* mine_row = mine + (my_row < rows ? my_row * 64 + quad * 16 : 0);

    struct Held {
        uintx4 code[NT];
        GroupValues<GPB, WIDE> s[NT], z[NT];
    } held[DEPTH];
    constexpr int X_SETS = GPB == 4 || MT == 2 ? 2 : DEPTH;   // four groups' scales or twice the rows leave registers for the next turn's x only
    BlockOfX<TYPE, REGS, MT> x[X_SETS];
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
    auto fetch_x = [&](int set, int block) {
        if (block < blocks) x[set].fetch(static_cast<const T*>(a.x), a.M, K, block, lane, my_row);
    };

    floatx4 acc[MT][NT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) acc[mt][nt] = floatx4{0, 0, 0, 0};
    uintx4 ones;
#pragma unroll
    for (int i = 0; i < 4; ++i) ones[i] = Codes<TYPE>::ONES;

    auto multiply = [&](const Held& h, const BlockOfX<TYPE, REGS, MT>& bx) {
        bx.to_lds(mine, lane);
#pragma unroll
        for (int g = 0; g < GPB; ++g) {
            floatx4 p[MT][NT], sum[MT];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                sum[mt] = floatx4{0, 0, 0, 0};
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) p[mt][nt] = floatx4{0, 0, 0, 0};
            }
#pragma unroll
            for (int i = g * SG; i < (g + 1) * SG; ++i) {
                uintx4 xa[MT];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    xa[mt] = bx.operand(mt, i, mine_row, my_row + 16 * mt < rows);
                    sum[mt] = Codes<TYPE>::mfma(xa[mt], ones, sum[mt]);
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const uintx4 codes = unpack_codes<TYPE>(h.code[nt][i]);
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) p[mt][nt] = Codes<TYPE>::mfma(xa[mt], codes, p[mt][nt]);
                }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const float s = h.s[nt].at(g, half), z = a.with_zeros ? h.z[nt].at(g, half) : 8.f;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int r = 0; r < REGS; ++r) acc[mt][nt][r] = __builtin_fmaf(s, __builtin_fmaf(-z, sum[mt][r], p[mt][nt][r]), acc[mt][nt][r]);
            }
            if (GPB == 4) __builtin_amdgcn_sched_barrier(0);   // all groups' codes unpacked at once have no room in registers
        }
    };

#pragma unroll
    for (int d = 0; d < DEPTH; ++d) fetch(held[d]);
#pragma unroll
    for (int d = 0; d < X_SETS - 1; ++d) fetch_x(d, wave + d * waves);
    for (int block = wave; block < blocks;) {
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            if (block < blocks) {
                fetch_x((d + X_SETS - 1) % X_SETS, block + (X_SETS - 1) * waves);
                multiply(held[d], x[d % X_SETS]);
                fetch(held[d]);
            }
            block += waves;
        }
    }

    // the waves' sums side by side in LDS, then one thread per result: waves and pieces in order
    __syncthreads();
    float* red = reinterpret_cast<float*>(lds);
    constexpr int WIDTH = NT * 16;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int r = 0; r < REGS; ++r) {
                const int row = mt * 16 + r * 4 + quad;
                if (row < rows) red[(wave * rows + row) * WIDTH + nt * 16 + col] = acc[mt][nt][r];
            }
    __syncthreads();
    for (int i = threadIdx.x; i < a.M * WIDTH; i += blockDim.x) {
        const int m = i / WIDTH, c = i - m * WIDTH, n = tile0 * 16 + c;
        if (n >= a.lay.N) continue;
        float v = 0;
        for (int w = 0; w < waves; ++w)
#pragma unroll
            for (int p = 0; p < PIECES; ++p) v += red[(w * rows + m * PIECES + p) * WIDTH + c];
        v *= 1 / Codes<TYPE>::UNIT;
        if (a.bias) v += (float)static_cast<const T*>(a.bias)[n];
        static_cast<T*>(a.y)[(size_t)m * a.lay.N + n] = (T)v;
    }
}

template <int TYPE, int GPB>
hipError_t stream_launch(const StreamArgs& a, hipStream_t stream)
{
    const int rows = a.M * pieces_of<TYPE>();
    // two tiles a workgroup share x and its column sums, as soon as that leaves a workgroup for every compute unit
    const int nt = a.lay.tiles >= 512 ? 2 : 1;
    int waves = nt == 1 && rows <= 16 ? 16 : 8;
    while (waves > 1 && waves / 2 >= a.lay.blocks) waves /= 2;
    // the waves' sums; before that, of a 32-bit x, their blocks of pieces
    const size_t own = TYPE == CAKE_HIP_F32 ? (rows <= 4 ? 3 : rows <= 16 ? 15 : 30) * 256 : 0;
    const size_t lds = waves * std::max((size_t)rows * nt * 64, own);
    const dim3 grid((a.lay.tiles + nt - 1) / nt), block(64 * waves);
    auto run = [&](auto kernel) {
        kernel<<<grid, block, lds, stream>>>(a);
        return hipGetLastError();
    };
    auto of_width = [&](auto wide) {
        constexpr bool W = decltype(wide)::value;
        if (rows <= 4) return nt == 1 ? run(&linear_q4_stream_kernel<TYPE, GPB, W, 1, 1, 1>) : run(&linear_q4_stream_kernel<TYPE, GPB, W, 1, 2, 1>);
        if (rows <= 16) return nt == 1 ? run(&linear_q4_stream_kernel<TYPE, GPB, W, 4, 1, 1>) : run(&linear_q4_stream_kernel<TYPE, GPB, W, 4, 2, 1>);
        return nt == 1 ? run(&linear_q4_stream_kernel<TYPE, GPB, W, 4, 1, 2>) : run(&linear_q4_stream_kernel<TYPE, GPB, W, 4, 2, 2>);
    };
    return a.lay.scale_type == CAKE_HIP_F32 ? of_width(std::true_type()) : of_width(std::false_type());
}

// What fits two tiles of 16 rows of pieces is streamed: one launch instead of three (17 rows of 4096 x 4096 9.8 us,
// in a band 15.9; of 14336 x 4096 in groups of 32 21 and 34; 10 of fp32 12 and 20).  Every workgroup reads all of x
// itself, though, and with more than 24 rows of many columns that costs more (32 rows of 4096 x 14336 30 and
// 27, of 16384 x 16384 71 and 63, but of 4096 x 4096 12 and 16).
bool streams(int M, int K, int type) { return type == CAKE_HIP_F32 ? M <= 10 : M <= 24 || (M <= 32 && K <= 8192); }

}  // namespace

size_t linear_q4_workspace(int M, int N, int K, int type)
{
    return M == 0 || N == 0 || streams(M, K, type) ? 0 : linear_q4_bands_workspace(M, N, K, type);
}

hipError_t launch_linear_q4(const void* x, const void* q, const void* bias, void* y, int type, int M, const Q4Layout& lay,
                            bool with_zeros, void* workspace, hipStream_t stream)
{
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
        q4_for_type_and_group(type, lay.groups_per_block,
                              [&](auto t, auto gpb) { e = stream_launch<decltype(t)::value, decltype(gpb)::value>(a, stream); });
        return e;
    }
    return launch_linear_q4_bands(x, q, bias, y, type, M, lay, with_zeros, workspace, stream);
}

}  // namespace cake
