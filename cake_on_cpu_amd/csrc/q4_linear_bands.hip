// q4_linear_bands.hip -- y[M][N] = x[M][K] . v[N][K]^T (+ bias) with v in 4 bits for many rows of x.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "kernels.hpp"
#include "q4_operands.hpp"

namespace cake {

namespace {

// A stage of the product is 64 columns of x (32 of an fp32 x, whose three pieces take their room), a
// band is 2 MTW tiles of 16 rows.  A band's stage is one record: the tiles as A operands, 1 KB per
// tile, step of 32 columns and piece, and behind them for every run of columns under one scale the rows'
// sums (times -8 where there are no zero points).
template <int TYPE, int GROUPS_, int MTW>
struct Record {
    static constexpr int PIECES = pieces_of<TYPE>();
    static constexpr int STEPS = TYPE == CAKE_HIP_F32 ? 1 : 2;
    static constexpr int GROUPS = GROUPS_;   // runs of columns under one scale in a stage: 2 for 16-bit x and groups of 32, else 1
    static constexpr int TILES = 2 * MTW;
    static constexpr int OPERANDS = TILES * STEPS * PIECES;                 // KB
    static constexpr int SUMS = (TILES * 16 * GROUPS * 4 + 1023) / 1024;    // KB
    static constexpr int KB = (OPERANDS + SUMS + 7) / 8 * 8;                 // whole rounds of eight waves
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

// x into records: a wave per tile and stage.
template <int TYPE, int GROUPS, int MTW, bool ZEROS>
__global__ __launch_bounds__(256) void linear_q4_records_kernel(BandArgs a)
{
    typedef typename Element<TYPE>::T T;
    typedef Record<TYPE, GROUPS, MTW> R;
    const int lane = threadIdx.x & 63;
    const size_t unit = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int tile = (int)(unit % R::TILES);
    const size_t record = unit / R::TILES;
    if (record >= (size_t)a.bands * a.stages) return;
    const int band = (int)(record / a.stages), stage = (int)(record - (size_t)band * a.stages);
    const int row = (band * R::TILES + tile) * 16 + (lane & 15);
    unsigned char* to = a.records + record * (R::KB * 1024);
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
        for (int e = 0; e < 8; ++e) sum += (float)v[e];
        if (i + 1 == R::STEPS || GROUPS == R::STEPS) {   // the end of a run
            sum += __shfl_xor(sum, 16);
            sum += __shfl_xor(sum, 32);
            const int g = GROUPS == 1 ? 0 : i;
            if (lane < 16)
                reinterpret_cast<float*>(to + R::OPERANDS * 1024)[(g * R::TILES + tile) * 16 + lane] = ZEROS ? sum : -8.f * sum;
            sum = 0;
        }
    }
}

// y for bands of 32 MTW rows of x and strips of 256 rows of v: 2 x 4 waves of MTW x 4 tiles each.  A
// band's records pass through LDS, two stages deep; codes go from memory to the registers of the wave that
// multiplies them.  Per run of columns the matrix pipe starts from -8 times the rows' sums (or from zero,
// and the zero point is applied behind it) and what comes out is scaled and added: for 16-bit x
// one scaling per 2 matrix instructions (per 1 with groups of 32), which still fits beside them.
template <int TYPE, int GROUPS, int MTW, bool ZEROS>
__global__ __launch_bounds__(512, 2) void linear_q4_band_kernel(BandArgs a)
{
    typedef typename Element<TYPE>::T T;
    typedef Record<TYPE, GROUPS, MTW> R;
    constexpr int NT = 4, LOADS = R::KB / 8, RUN = R::STEPS / GROUPS;
    extern __shared__ __align__(16) unsigned char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int quad = lane >> 4, col = lane & 15;
    const int wm = wave >> 2, wn = wave & 3;
    const int bands = a.bands, strips = (a.lay.tiles + 15) / 16;
    // bands of one strip run together, and with a multiple of eight of them each die keeps its band's x
    const int slice = (int)(blockIdx.x / (unsigned)(bands * strips)), id = (int)(blockIdx.x - (unsigned)slice * (unsigned)(bands * strips));
    const int strip = id / bands, band = id - strip * bands;
    const int s0 = (int)((long long)a.stages * slice / a.slices), s1 = (int)((long long)a.stages * (slice + 1) / a.slices);

    const unsigned char* from = a.records + ((size_t)band * a.stages + s0) * (R::KB * 1024);
    uintx4 next[LOADS];
    auto fetch = [&](int l) {
        next[l] = *reinterpret_cast<const uintx4*>(from + (unsigned)((l * 8 + wave) * 1024 + lane * 16));
    };
    auto put = [&](int l, int to) {
        *reinterpret_cast<uintx4*>(lds + to * (R::KB * 1024) + (l * 8 + wave) * 1024 + lane * 16) = next[l];
    };
    // Codes and scales of a stage, as they lie: scalar addresses and a lane's place behind them.  A
    // 16-bit scale is fetched as the word that holds it and taken out where it is used, so that
    // nothing waits for it here and no branch over its type breaks the loop into pieces.
    const int gpb = a.lay.groups_per_block;
    const bool wide = a.lay.scale_type == CAKE_HIP_F32, half = a.lay.scale_type == CAKE_HIP_F16;
    const int scale_bytes = wide ? 4 : 2;
    unsigned code[NT][R::STEPS], s[NT][GROUPS], z[NT][GROUPS];
    auto group_of = [&](int stage, int g) { return stage * R::STEPS % 4 * gpb / 4 + g; };
    auto fetch_codes = [&](int stage) {
        const int block = stage * R::STEPS / 4, i0 = stage * R::STEPS % 4;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int tile = min(strip * 16 + wn * NT + nt, a.lay.tiles - 1);
            const size_t unit = (size_t)tile * a.lay.blocks + block;
            const unsigned char* at = a.q + unit * 1024 + i0 * 4;
            if (R::STEPS == 2) {
                const uintx2 two = *reinterpret_cast<const uintx2*>(at + (unsigned)lane * 16);
#pragma unroll
                for (int i = 0; i < R::STEPS; ++i) code[nt][i] = two[i & 1];
            } else {
                code[nt][0] = *reinterpret_cast<const unsigned*>(at + (unsigned)lane * 16);
            }
            const unsigned char* scales = a.q + a.lay.scales_at + unit * (16 * gpb * scale_bytes);
            const unsigned char* zeros = a.q + a.lay.zeros_at + unit * (16 * gpb * scale_bytes);
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) {
                const unsigned byte = (unsigned)(col * gpb + group_of(stage, g)) * scale_bytes & ~3u;
                s[nt][g] = *reinterpret_cast<const unsigned*>(scales + byte);
                z[nt][g] = ZEROS ? *reinterpret_cast<const unsigned*>(zeros + byte) : 0u;
            }
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
        for (int l = 0; l < LOADS; ++l) fetch(l);
        fetch_codes(s0);
#pragma unroll
        for (int l = 0; l < LOADS; ++l) put(l, 0);
        if (s0 + 1 < s1) from += R::KB * 1024;
#pragma unroll
        for (int l = 0; l < LOADS; ++l) fetch(l);
    }
    __syncthreads();
    for (int stage = s0; stage < s1; ++stage) {
        const int now = (stage - s0) & 1;
        const unsigned char* at = lds + now * (R::KB * 1024);
        if (stage + 2 < s1) from += R::KB * 1024;
        uintx4 b[NT][R::STEPS];
        float now_s[NT][GROUPS], now_z[NT][GROUPS];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int i = 0; i < R::STEPS; ++i) b[nt][i] = unpack_codes<TYPE>(code[nt][i]);
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) {
                now_s[nt][g] = scale_in(s[nt][g], group_of(stage, g));
                now_z[nt][g] = ZEROS ? scale_in(z[nt][g], group_of(stage, g)) : 0.f;
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        fetch_codes(stage + 1 < s1 ? stage + 1 : stage);   // past the last stage: fetched again, not used
        // operands one tile ahead of the products; the compiler left alone reads them all at the start
        // and has no registers left
        uintx4 xa[2][R::STEPS][R::PIECES];
        floatx4 sum[2][GROUPS];
        auto read = [&](int mt) {
            const int tile = wm * MTW + mt;
#pragma unroll
            for (int i = 0; i < R::STEPS; ++i)
#pragma unroll
                for (int p = 0; p < R::PIECES; ++p)
                    xa[mt & 1][i][p] = *reinterpret_cast<const uintx4*>(at + ((tile * R::STEPS + i) * R::PIECES + p) * 1024 + lane * 16);
#pragma unroll
            for (int g = 0; g < GROUPS; ++g)
                sum[mt & 1][g] = *reinterpret_cast<const floatx4*>(at + R::OPERANDS * 1024 + ((g * R::TILES + tile) * 16 + quad * 4) * 4);
        };
        read(0);
#pragma unroll
        for (int mt = 0; mt < MTW; ++mt) {
            if (mt + 1 < MTW) read(mt + 1);
            // this tile's share of the next stage: out of the registers, and the stage after it in
#pragma unroll
            for (int l = mt * LOADS / MTW; l < (mt + 1) * LOADS / MTW; ++l) {
                put(l, now ^ 1);
                fetch(l);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) {
                floatx4 p[NT];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) p[nt] = ZEROS ? floatx4{0, 0, 0, 0} : sum[mt & 1][g];
#pragma unroll
                for (int i = g * RUN; i < (g + 1) * RUN; ++i)
#pragma unroll
                    for (int piece = R::PIECES - 1; piece >= 0; --piece)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) p[nt] = Codes<TYPE>::mfma(xa[mt & 1][i][piece], b[nt][i], p[nt]);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        acc[mt][nt][r] = __builtin_fmaf(now_s[nt][g], ZEROS ? __builtin_fmaf(-now_z[nt][g], sum[mt & 1][g][r], p[nt][r]) : p[nt][r],
                                                        acc[mt][nt][r]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        __syncthreads();
    }

#pragma unroll
    for (int mt = 0; mt < MTW; ++mt) {
        const int m = ((band * 2 + wm) * MTW + mt) * 16 + quad * 4;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int n = (strip * 16 + wn * NT + nt) * 16 + col;
            if (n >= a.lay.N) continue;
            if (a.partial) {
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (m + r < a.M) a.partial[((size_t)slice * a.M + m + r) * a.lay.N + n] = acc[mt][nt][r];
            } else {
                const float bias = a.bias ? (float)static_cast<const T*>(a.bias)[n] : 0.f;
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (m + r < a.M) static_cast<T*>(a.y)[(size_t)(m + r) * a.lay.N + n] = (T)(acc[mt][nt][r] + bias);
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
    int mtw, bands, stages, slices;
    size_t record_bytes, bytes;
};

BandPlan band_plan(int M, int N, int K, int type)
{
    BandPlan p;
    // time of a band next to one of 256 rows: a narrow one leaves the matrix pipe idle behind its codes
    const float cost[3] = {0.40f, 0.60f, 1.f};
    float least = 0;
    for (int i = 0; i < 3; ++i) {
        const int rows = 64 << i;
        const float time = cost[i] * (float)((M + (long long)rows - 1) / rows);
        if (i == 0 || time < least) {
            least = time;
            p.mtw = 2 << i;
        }
    }
    const int rows = 32 * p.mtw, steps = type == CAKE_HIP_F32 ? 1 : 2;
    p.bands = (int)((M + (long long)rows - 1) / rows);
    p.stages = (int)(((long long)K + 127) / 128) * (4 / steps);
    const long long groups = (((long long)N + 255) / 256) * p.bands;
    // slices of K, of eight stages at least, until every compute unit has a workgroup
    p.slices = 1;
    while (groups * (p.slices + 1) <= 256 && p.stages / (p.slices + 1) >= 8) ++p.slices;
    // the largest record of the type: two runs a stage
    const int kb = (2 * p.mtw * steps * (type == CAKE_HIP_F32 ? 3 : 1) + (2 * p.mtw * 16 * 2 * 4 + 1023) / 1024 + 7) / 8 * 8;
    p.record_bytes = (size_t)p.bands * p.stages * kb * 1024;
    p.bytes = p.record_bytes + (p.slices > 1 ? (size_t)p.slices * M * N * sizeof(float) : 0);
    return p;
}

template <int TYPE, int GROUPS, int MTW, bool ZEROS>
hipError_t band_launch(const BandArgs& a, hipStream_t stream)
{
    typedef Record<TYPE, GROUPS, MTW> R;
    const size_t units = (size_t)a.bands * a.stages * R::TILES;
    hipError_t e = hipSuccess;
    if (units) {   // (K == 0 is only a bias)
        linear_q4_records_kernel<TYPE, GROUPS, MTW, ZEROS><<<(unsigned)((units + 3) / 4), 256, 0, stream>>>(a);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    constexpr size_t LDS = (size_t)2 * R::KB * 1024;
    auto kernel = &linear_q4_band_kernel<TYPE, GROUPS, MTW, ZEROS>;
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

template <int TYPE, int GROUPS>
hipError_t bands_launch(const BandArgs& a, int mtw, bool zeros, hipStream_t stream)
{
    if (mtw == 2) return zeros ? band_launch<TYPE, GROUPS, 2, true>(a, stream) : band_launch<TYPE, GROUPS, 2, false>(a, stream);
    if (mtw == 4) return zeros ? band_launch<TYPE, GROUPS, 4, true>(a, stream) : band_launch<TYPE, GROUPS, 4, false>(a, stream);
    return zeros ? band_launch<TYPE, GROUPS, 8, true>(a, stream) : band_launch<TYPE, GROUPS, 8, false>(a, stream);
}

}  // namespace

size_t linear_q4_bands_workspace(int M, int N, int K, int type) { return band_plan(M, N, K, type).bytes; }

hipError_t launch_linear_q4_bands(const void* x, const void* q, const void* bias, void* y, int type, int M, const Q4Layout& lay,
                                  bool with_zeros, void* workspace, hipStream_t stream)
{
    const BandPlan p = band_plan(M, lay.N, lay.K, type);
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
    const bool two = type != CAKE_HIP_F32 && lay.groups_per_block == 4;
    if (type == CAKE_HIP_F32) return bands_launch<CAKE_HIP_F32, 1>(a, p.mtw, with_zeros, stream);
    if (type == CAKE_HIP_F16)
        return two ? bands_launch<CAKE_HIP_F16, 2>(a, p.mtw, with_zeros, stream) : bands_launch<CAKE_HIP_F16, 1>(a, p.mtw, with_zeros, stream);
    return two ? bands_launch<CAKE_HIP_BF16, 2>(a, p.mtw, with_zeros, stream) : bands_launch<CAKE_HIP_BF16, 1>(a, p.mtw, with_zeros, stream);
}

}  // namespace cake
