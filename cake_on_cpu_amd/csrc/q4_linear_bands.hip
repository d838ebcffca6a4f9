// q4_linear_bands.hip -- y[M][N] = x[M][K] . v[N][K]^T (+ bias) with v in 4 bits for many rows of x.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "kernels.hpp"
#include "q4_operands.hpp"

namespace cake {

namespace {

// A band is 64, 128 or 256 rows of x.  A stage of the product is a block of 128 columns, or what of it
// fits LDS twice where three pieces of an fp32 x take their room.  A band's stage is one record: its
// tiles of 16 rows as A operands, 1 KB per tile, step of 32 columns and piece, and behind them for every
// run of columns under one scale the rows' sums: times -8 where there are no zero points, where the
// matrix pipe then starts a run; with zero points as three bf16 pieces, of which one more matrix
// instruction a stage makes the sum over its runs of s z sum(x) -- eight products of pieces each, all but
// the last pieces' own, below 2^-30 -- and takes it from the result.  (Taken from each run's sum instead, at
// one operation an element beside the scaling's one, 2048 rows of 14336 x 4096 in groups of 32 took 526 us
// for 405.)
// Eight waves share the strip of 256 rows of v that a workgroup multiplies a band with.  Each takes 32
// of them and all the band, so that no code is unpacked twice: unpacking and scaling take the vector
// pipe 180 instructions a stage (groups of 128, 256 rows) beside 128 of the matrix pipe, and those that
// two waves repeat, or that scale after every 64 columns, cost as much time as they take (2 x 4 waves,
// 64 columns: 283 us for 2048 rows, 14336 x 4096; 226 this way).
template <int TYPE, int GROUPS_, int ROWS_, bool ZEROS>
struct Record {
    static constexpr int ROWS = ROWS_;
    static constexpr int PIECES = pieces_of<TYPE>();
    static constexpr int STEPS = TYPE == CAKE_HIP_F32 ? 256 / ROWS : 4;
    static constexpr int GROUPS = GROUPS_;                                  // runs of columns under one scale in a stage: a step each for groups of 32, ...
    static constexpr int NT = 2;                                            // a wave's tiles of the strip
    static constexpr int TILES = ROWS / 16;
    static constexpr int OPERANDS = TILES * STEPS * PIECES;                 // KB
    static constexpr int SUMS = ROWS * GROUPS;                              // of 4 bytes, or 16 of pieces
    static constexpr int BYTES = OPERANDS * 1024 + SUMS * (ZEROS ? 16 : 4);
    // stages that codes are fetched ahead: those of a narrow band are over before memory answers
    static constexpr int CODES_AHEAD = ROWS == 256 ? 1 : 2;
};

struct BandArgs {
    const void* x;
    const unsigned char* q;
    const void* bias;
    void* y;
    unsigned char* records;
    float* partial;       // [slice][M][N], or nullptr
    Q4Layout lay;
    int M, bands, stages, slices;
};

// The pieces of v in the order of the products: which piece (0 leading, 1 middle, 2 last) each of the eight slots takes
struct PieceOrder { int of[8]; };
constexpr PieceOrder SUM_PIECES = {{0, 0, 1, 1, 0, 2, 1, 2}}, ZERO_PIECES = {{0, 1, 0, 1, 2, 0, 2, 1}};
__device__ __forceinline__ uintx4 eight_pieces(float v, PieceOrder order)
{
    unsigned piece[3];
#pragma unroll
    for (int p = 0; p < 3; ++p) {
        piece[p] = __builtin_bit_cast(unsigned, v) & 0xFFFF0000u;
        v -= __builtin_bit_cast(float, piece[p]);   // exact
    }
    uintx4 out;
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = piece[order.of[2 * i]] >> 16 | piece[order.of[2 * i + 1]];
    return out;
}

// x into records: a wave per tile and stage.
template <int TYPE, int GROUPS, int ROWS, bool ZEROS>
__global__ __launch_bounds__(256) void linear_q4_records_kernel(BandArgs a)
{
    typedef typename Element<TYPE>::T T;
    typedef Record<TYPE, GROUPS, ROWS, ZEROS> R;
    const int lane = threadIdx.x & 63;
    const size_t unit = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int tile = (int)(unit % R::TILES);
    const size_t record = unit / R::TILES;
    if (record >= (size_t)a.bands * a.stages) return;
    const int band = (int)(record / a.stages), stage = (int)(record - (size_t)band * a.stages);
    const int row = (band * R::TILES + tile) * 16 + (lane & 15);
    unsigned char* to = a.records + record * R::BYTES;
    float sum = 0;
#pragma unroll
    for (int i = 0; i < R::STEPS; ++i) {
        const int k = (stage * R::STEPS + i) * 32 + (lane >> 4) * 8;
        T v[8];
        load_eight<TYPE>(static_cast<const T*>(a.x) + (size_t)row * a.lay.K + k, row < a.M ? a.lay.K - k : 0, v);
#pragma unroll
        for (int p = 0; p < R::PIECES; ++p)
            *reinterpret_cast<uintx4*>(to + ((tile * R::STEPS + i) * R::PIECES + p) * 1024 + lane * 16) = piece_of<TYPE>(v, p);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum += (float)v[e] * Codes<TYPE>::UNIT;
        if ((i + 1) % (R::STEPS / GROUPS) == 0) {   // the end of a run
            sum += __shfl_xor(sum, 16);
            sum += __shfl_xor(sum, 32);
            const int g = i / (R::STEPS / GROUPS);
            if (lane < 16) {
                const int at = (g * R::TILES + tile) * 16 + lane;
                if (ZEROS) reinterpret_cast<uintx4*>(to + R::OPERANDS * 1024)[at] = eight_pieces(sum, SUM_PIECES);
                else reinterpret_cast<float*>(to + R::OPERANDS * 1024)[at] = -8.f * sum;
            }
            sum = 0;
        }
    }
}

// y for bands of x and strips of 256 rows of v.  A band's records pass through LDS, two stages deep, by way of
// registers; codes go from memory to the registers of the wave that multiplies them.  Per run of
// columns the matrix pipe starts from -8 times the rows' sums (or from zero, and the zero point is
// applied behind it) and what comes out is scaled and added while the next run is multiplied.
template <int TYPE, int GROUPS, int ROWS, bool ZEROS>
__global__ __launch_bounds__(512, 2) void linear_q4_band_kernel(BandArgs a)
{
    typedef typename Element<TYPE>::T T;
    typedef Record<TYPE, GROUPS, ROWS, ZEROS> R;
    constexpr int NT = R::NT, MTW = R::TILES, STEPS = R::STEPS, PIECES = R::PIECES, RUN = STEPS / GROUPS, SETS = R::CODES_AHEAD;
    // A record is fetched in LOADS rounds of 8 KB, an even number.  Round l is put into LDS beside tile slot(l) of the stage
    // before its own and fetched AHEAD tiles earlier, half a stage, so that half of the rounds are in registers.
    static_assert(R::OPERANDS % 16 == 0, "two halves of whole rounds");
    constexpr int LOADS = R::OPERANDS / 8, AHEAD = MTW / 2, HELD = LOADS / 2;
    constexpr int SUM_LOADS = (R::SUMS + 511) / 512;
    extern __shared__ __align__(16) unsigned char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int quad = lane >> 4, col = lane & 15;
    const int bands = a.bands, strips = (a.lay.tiles + 15) / 16;
    // bands of one strip run together, and with a multiple of eight of them each die keeps its band's x
    const int slice = (int)(blockIdx.x / (unsigned)(bands * strips)), id = (int)(blockIdx.x - (unsigned)slice * (unsigned)(bands * strips));
    const int strip = id / bands, band = id - strip * bands;
    const int s0 = (int)((long long)a.stages * slice / a.slices), s1 = (int)((long long)a.stages * (slice + 1) / a.slices);

    const unsigned char* records = a.records + (size_t)band * a.stages * R::BYTES;
    auto record_of = [&](int stage) { return records + (size_t)min(stage, s1 - 1) * R::BYTES; };   // past the last: fetched again, not used
    auto slot = [](int l) { return l * MTW / LOADS; };
    auto part = [&](int l) { return l * 8 + wave; };
    uintx4 next[HELD];
    typedef typename std::conditional<ZEROS, uintx4, float>::type Sum;
    Sum next_sum[SUM_LOADS];
    auto fetch = [&](int l, const unsigned char* from) {
        next[l % HELD] = *reinterpret_cast<const uintx4*>(from + (unsigned)(part(l) * 1024 + lane * 16));
    };
    auto put = [&](int l, int to) {
        *reinterpret_cast<uintx4*>(lds + to * R::BYTES + part(l) * 1024 + lane * 16) = next[l % HELD];
    };
    auto fetch_sums = [&](const unsigned char* from) {
#pragma unroll
        for (int i = 0; i < SUM_LOADS; ++i) next_sum[i] = reinterpret_cast<const Sum*>(from + R::OPERANDS * 1024)[min(i * 512 + (int)threadIdx.x, R::SUMS - 1)];
    };
    auto put_sums = [&](int to) {
#pragma unroll
        for (int i = 0; i < SUM_LOADS; ++i) reinterpret_cast<Sum*>(lds + to * R::BYTES + R::OPERANDS * 1024)[min(i * 512 + (int)threadIdx.x, R::SUMS - 1)] = next_sum[i];
    };

    // Codes and scales of a stage, as they lie: scalar addresses and a lane's place behind them.  A
    // 16-bit scale is fetched as the word that holds it and taken out where it is used, so that
    // nothing waits for it here and no branch over its type breaks the loop into pieces.
    const int gpb = a.lay.groups_per_block;
    const bool wide = a.lay.scale_type == CAKE_HIP_F32, half = a.lay.scale_type == CAKE_HIP_F16;
    const int scale_bytes = wide ? 4 : 2;
    unsigned code[SETS][NT][STEPS], s[SETS][NT][GROUPS], z[SETS][NT];
    auto group_of = [&](int stage, int g) { return stage * STEPS % 4 * gpb / 4 + g; };
    auto fetch_codes = [&](int set, int stage) {
        stage = min(stage, s1 - 1);   // past the last: fetched again, not used
        const int block = stage * STEPS / 4, i0 = stage * STEPS % 4;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int tile = min(strip * 16 + wave * NT + nt, a.lay.tiles - 1);
            const size_t unit = (size_t)tile * a.lay.blocks + block;
            __builtin_memcpy(code[set][nt], a.q + unit * 1024 + i0 * 4 + (unsigned)lane * 16, STEPS * 4);
            const unsigned char* scales = a.q + a.lay.scales_at + unit * (16 * gpb * scale_bytes);
            const unsigned char* zeros = a.q + a.lay.zeros_at + unit * (16 * gpb * scale_bytes);
#pragma unroll
            for (int g = 0; g < GROUPS; ++g)
                s[set][nt][g] = *reinterpret_cast<const unsigned*>(scales + ((unsigned)(col * gpb + group_of(stage, g)) * scale_bytes & ~3u));
            // the lane's quarter of the columns stands for a run of its own there
            z[set][nt] = ZEROS ? *reinterpret_cast<const unsigned*>(zeros + ((unsigned)(col * gpb + group_of(stage, quad % GROUPS)) * scale_bytes & ~3u)) : 0u;
        }
    };
    auto scale_in = [&](unsigned word, int group) {
        const unsigned narrow = word >> ((col * gpb + group & 1) * 16) & 0xFFFFu;
        const float f16 = (float)__builtin_bit_cast(_Float16, (unsigned short)narrow), bf16 = __builtin_bit_cast(float, narrow << 16);
        return wide ? __builtin_bit_cast(float, word) : half ? f16 : bf16;
    };

    floatx4 acc[MTW][NT];
#pragma unroll
    for (int mt = 0; mt < MTW; ++mt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) acc[mt][nt] = floatx4{0, 0, 0, 0};
    if (s0 < s1) {
#pragma unroll
        for (int d = 0; d < SETS; ++d) fetch_codes(d, s0 + d);
        fetch_sums(record_of(s0));
#pragma unroll
        for (int l0 = 0; l0 < LOADS; l0 += HELD) {
#pragma unroll
            for (int l = l0; l < l0 + HELD; ++l) fetch(l, record_of(s0));
#pragma unroll
            for (int l = l0; l < l0 + HELD; ++l) put(l, 0);
        }
        put_sums(0);
        fetch_sums(record_of(s0 + 1));
#pragma unroll
        for (int l = 0; l < HELD; ++l) fetch(l, record_of(s0 + 1));
    }
    __syncthreads();
    auto multiply = [&](int stage, int set) {
        const int now = (stage - s0) & 1;
        const unsigned char* at = lds + now * R::BYTES + lane * 16;
        const unsigned char* at_sums = lds + now * R::BYTES + R::OPERANDS * 1024 + (ZEROS ? (quad % GROUPS * R::TILES * 16 + col) * 16 : quad * 16);
        const unsigned char *from1 = record_of(stage + 1), *from2 = record_of(stage + 2);
        uintx4 b[NT][STEPS];
        float now_s[NT][GROUPS];
        uintx4 bz[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int i = 0; i < STEPS; ++i) b[nt][i] = unpack_codes<TYPE>(code[set][nt][i]);
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) now_s[nt][g] = scale_in(s[set][nt][g], group_of(stage, g));
            if (ZEROS) {
                float own = now_s[nt][0];
#pragma unroll
                for (int g = 1; g < GROUPS; ++g) own = quad == g ? now_s[nt][g] : own;
                own *= -scale_in(z[set][nt], group_of(stage, quad % GROUPS));
                bz[nt] = eight_pieces(quad < GROUPS ? own : 0.f, ZERO_PIECES);
            }
        }
        put_sums(now ^ 1);
        __builtin_amdgcn_sched_barrier(0);
        fetch_codes(set, stage + SETS);
        fetch_sums(from2);
        // Operands are read one tile ahead of their products, into the registers that the step before has
        // just left; the compiler left alone reads them all at the start and has no registers for it.
        auto operand = [&](int mt, int i, int p) {
            return *reinterpret_cast<const uintx4*>(at + ((mt * STEPS + i) * PIECES + p) * 1024);
        };
        // without zero points four rows' sums of a run, with them the pieces of the lane's row and quarter
        auto sums_of = [&](int mt, int g) {
            return *reinterpret_cast<const floatx4*>(at_sums + (ZEROS ? mt * 256 : (g * R::TILES + mt) * 64));
        };
        uintx4 xa[STEPS][PIECES];
#pragma unroll
        for (int i = 0; i < STEPS; ++i)
#pragma unroll
            for (int p = 0; p < PIECES; ++p) xa[i][p] = operand(0, i, p);
        floatx4 coming = sums_of(0, 0), p[2][NT];
        auto add = [&](int mt, int g) {
            const int turn = (mt * GROUPS + g) & 1;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    acc[mt][nt][r] = __builtin_fmaf(now_s[nt][g], p[turn][nt][r], acc[mt][nt][r]);
        };
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int mt = 0; mt < MTW; ++mt) {
#pragma unroll
            for (int l = 0; l < LOADS; ++l)
                if (slot(l) == mt) put(l, now ^ 1);
#pragma unroll
            for (int l = 0; l < LOADS; ++l)
                if (slot(l) == (mt + AHEAD) % MTW) fetch(l, mt < AHEAD ? from1 : from2);
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) {
                const int turn = (mt * GROUPS + g) & 1;
                const floatx4 sums = coming;
                if (!ZEROS && g + 1 < GROUPS) coming = sums_of(mt, g + 1);
                else if (g + 1 == GROUPS && mt + 1 < MTW) coming = sums_of(mt + 1, 0);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) p[turn][nt] = ZEROS ? floatx4{0, 0, 0, 0} : sums;
                if (ZEROS && g + 1 == GROUPS) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        acc[mt][nt] = Codes<CAKE_HIP_BF16>::mfma(__builtin_bit_cast(uintx4, sums), bz[nt], acc[mt][nt]);
                }
#pragma unroll
                for (int i = g * RUN; i < (g + 1) * RUN; ++i)
#pragma unroll
                    for (int piece = PIECES - 1; piece >= 0; --piece) {
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) p[turn][nt] = Codes<TYPE>::mfma(xa[i][piece], b[nt][i], p[turn][nt]);
                        if (mt + 1 < MTW) xa[i][piece] = operand(mt + 1, i, piece);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                // the run before this one, whose products are done
                if (g > 0) add(mt, g - 1);
                else if (mt > 0) add(mt - 1, GROUPS - 1);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        add(MTW - 1, GROUPS - 1);
        __syncthreads();
    };
    for (int stage = s0; stage < s1; stage += SETS) {
        multiply(stage, 0);
        if (SETS == 2 && stage + 1 < s1) multiply(stage + 1, SETS - 1);
    }

#pragma unroll
    for (int mt = 0; mt < MTW; ++mt) {
        const int m = (band * MTW + mt) * 16 + quad * 4;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int n = (strip * 16 + wave * NT + nt) * 16 + col;
            if (n >= a.lay.N) continue;
            if (a.partial) {
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (m + r < a.M) a.partial[((size_t)slice * a.M + m + r) * a.lay.N + n] = acc[mt][nt][r] * (1 / Codes<TYPE>::UNIT);
            } else {
                const float bias = a.bias ? (float)static_cast<const T*>(a.bias)[n] : 0.f;
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (m + r < a.M) static_cast<T*>(a.y)[(size_t)(m + r) * a.lay.N + n] = (T)(acc[mt][nt][r] * (1 / Codes<TYPE>::UNIT) + bias);
            }
        }
    }
}

// The slices of y added up in order.
template <int TYPE>
__global__ __launch_bounds__(256) void linear_q4_join_kernel(BandArgs a)
{
    typedef typename Element<TYPE>::T T;
    const size_t all = (size_t)a.M * a.lay.N;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (size_t)gridDim.x * 256) {
        float v = a.partial[i];
        for (int s = 1; s < a.slices; ++s) v += a.partial[s * all + i];
        if (a.bias) v += (float)static_cast<const T*>(a.bias)[i % a.lay.N];
        static_cast<T*>(a.y)[i] = (T)v;
    }
}

// How a product of many rows is cut: rows per band, slices of K, and the workspace's parts.
struct BandPlan {
    int rows, bands, stages, slices;
    size_t record_bytes, bytes;
};

// Microseconds of 128 columns of a band on a busy device: under one run without zero points, more for every further
// run, and with zero points (measured on 2048 rows of 14336 x 4096).  Bands of 256 rows need fewer passes
// over the codes, but neither the pieces of an fp32 x nor zero points leave them the registers: their
// spills cost more (281 us against 287 with zero points under groups of 128, 514 against 405 under groups
// of 32, fp32 692 to 1109 against 578 to 763 with 64 rows), and so they are only for 16-bit x without.
struct BandCost {
    int rows;
    float once, run, zeros;
};
constexpr BandCost BAND_COSTS[2][3] = {{{64, 1.29f, 0.26f, 0.25f}, {128, 1.95f, 0.31f, 0.28f}, {256, 3.5f, 0.8f, 0.f}},
                                       {{64, 2.58f, 0.2f, 0.23f}, {128, 5.f, 0.2f, 0.64f}, {0, 0.f, 0.f, 0.f}}};
enum { BAND_CUS = 256, BAND_MAX_SLICES = 24 };   // fixed, so that sizes alone decide on the workspace and the order of the sums

BandPlan band_plan(int M, int N, int K, int type, int groups_per_block, bool zeros)
{
    BandPlan best{};
    const int wide = type == CAKE_HIP_F32;
    const int blocks = (int)(((long long)K + 127) / 128);
    float least_us = 0;
    for (const BandCost& c : BAND_COSTS[wide]) {
        if (c.rows == 0 || (c.rows == 256 && zeros)) continue;
        const float block_us = c.once + c.run * (float)(groups_per_block - 1) + (zeros ? c.zeros : 0.f);
        const int bands = (int)((M + (long long)c.rows - 1) / c.rows);
        const long long groups = (((long long)N + 255) / 256) * bands;
        for (int s = 1; s <= BAND_MAX_SLICES && (s == 1 || (groups * s <= 2 * BAND_CUS && s <= blocks)); ++s) {
            const float rounds = (float)((groups * s + BAND_CUS - 1) / BAND_CUS);
            // a workgroup's beginning and end, and for slices another launch and a pass over their sums
            float us = rounds * (block_us * (float)((blocks + s - 1) / s) + 3.f);
            if (s > 1) us += 3.f + (float)s * (float)M * (float)N * 8 / 6e6f;
            if (best.rows == 0 || us < least_us) {
                least_us = us;
                best.rows = c.rows;
                best.bands = bands;
                best.slices = s;
            }
        }
    }
    best.stages = blocks * (wide ? best.rows / 64 : 1);
    // the largest record of the type: a run with pieces for each step of 32 columns
    const size_t steps = wide ? 256 / best.rows : 4, record = (size_t)best.rows * steps * (32 * 2 * (wide ? 3 : 1) + 16);
    best.record_bytes = ((size_t)best.bands * best.stages * record + 255) & ~(size_t)255;
    best.bytes = best.record_bytes + (best.slices > 1 ? (size_t)best.slices * M * N * sizeof(float) : 0);
    return best;
}

template <int TYPE, int GROUPS, int ROWS, bool ZEROS>
hipError_t band_launch(const BandArgs& a, hipStream_t stream)
{
    typedef Record<TYPE, GROUPS, ROWS, ZEROS> R;
    const size_t units = (size_t)a.bands * a.stages * R::TILES;
    hipError_t e = hipSuccess;
    if (units) {   // (K == 0 is only a bias)
        linear_q4_records_kernel<TYPE, GROUPS, ROWS, ZEROS><<<(unsigned)((units + 3) / 4), 256, 0, stream>>>(a);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    constexpr size_t LDS = (size_t)2 * R::BYTES;
    auto kernel = &linear_q4_band_kernel<TYPE, GROUPS, ROWS, ZEROS>;
    if (LDS > 64 * 1024) {
        e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)LDS);
        if (e != hipSuccess) return e;
    }
    const unsigned groups = (unsigned)((a.lay.tiles + 15) / 16) * (unsigned)a.bands * (unsigned)a.slices;
    kernel<<<groups, 512, LDS, stream>>>(a);
    if ((e = hipGetLastError()) != hipSuccess || a.slices == 1) return e;
    const size_t all = (size_t)a.M * a.lay.N;
    linear_q4_join_kernel<TYPE><<<(unsigned)std::min<size_t>((all + 255) / 256, 4096), 256, 0, stream>>>(a);
    return hipGetLastError();
}

template <int TYPE, int GROUPS, int ROWS>
hipError_t zeros_launch(const BandArgs& a, bool zeros, hipStream_t stream)
{
    if constexpr (ROWS < 256)
        if (zeros) return band_launch<TYPE, GROUPS, ROWS, true>(a, stream);
    return zeros ? hipErrorInvalidValue : band_launch<TYPE, GROUPS, ROWS, false>(a, stream);
}

template <int TYPE, int ROWS>
hipError_t rows_launch(const BandArgs& a, bool zeros, hipStream_t stream)
{
    constexpr int STEPS = Record<TYPE, 1, ROWS, false>::STEPS;
    const int groups = std::max(1, STEPS * a.lay.groups_per_block / 4);
    if (groups == 1) return zeros_launch<TYPE, 1, ROWS>(a, zeros, stream);
    if (groups == 2) return zeros_launch<TYPE, 2, ROWS>(a, zeros, stream);
    if constexpr (STEPS >= 4) return zeros_launch<TYPE, 4, ROWS>(a, zeros, stream);
    return hipErrorInvalidValue;
}

template <int TYPE>
hipError_t bands_launch(const BandArgs& a, int rows, bool zeros, hipStream_t stream)
{
    if (rows == 64) return rows_launch<TYPE, 64>(a, zeros, stream);
    if (rows == 128) return rows_launch<TYPE, 128>(a, zeros, stream);
    if constexpr (TYPE != CAKE_HIP_F32) return rows_launch<TYPE, 256>(a, zeros, stream);
    return hipErrorInvalidValue;
}

}  // namespace

size_t linear_q4_bands_workspace(int M, int N, int K, int type)
{
    size_t most = 0;   // whatever the weights' groups and zero points
    for (int per_block : {1, 2, 4})
        for (bool zeros : {false, true}) most = std::max(most, band_plan(M, N, K, type, per_block, zeros).bytes);
    return most;
}

hipError_t launch_linear_q4_bands(const void* x, const void* q, const void* bias, void* y, int type, int M, const Q4Layout& lay,
                                  bool with_zeros, void* workspace, hipStream_t stream)
{
    const BandPlan p = band_plan(M, lay.N, lay.K, type, lay.groups_per_block, with_zeros);
    BandArgs a{};
    a.x = x;
    a.q = static_cast<const unsigned char*>(q);
    a.bias = bias;
    a.y = y;
    a.records = static_cast<unsigned char*>(workspace);
    a.partial = p.slices > 1 ? reinterpret_cast<float*>(a.records + p.record_bytes) : nullptr;
    a.lay = lay;
    a.M = M;
    a.bands = p.bands;
    a.stages = p.stages;
    a.slices = p.slices;
    if (type == CAKE_HIP_F32) return bands_launch<CAKE_HIP_F32>(a, p.rows, with_zeros, stream);
    return type == CAKE_HIP_F16 ? bands_launch<CAKE_HIP_F16>(a, p.rows, with_zeros, stream) : bands_launch<CAKE_HIP_BF16>(a, p.rows, with_zeros, stream);
}

}  // namespace cake
