// orthogonalize.hip -- Newton-Schulz iterations on a batch of matrices:
//   x = g / (|g|_F + eps), then steps times  a = x x^T,  b = c1 a + c2 a a,  x = c0 x + b x
// (for more rows than columns on the transpose).
//
// All products run on the 16-bit matrix pipe at 32-bit accuracy.  A value v is kept as two fp16
// numbers, hi = fp16(v 2^e) and lo = fp16(v 2^e - hi): 11 significant bits each and the sign of lo
// leave at most 2^-23 of the value, and the power of two e keeps both parts in fp16's range (the
// iteration's values are bounded by its coefficients, so e is known beforehand).  A product is then
// hi hi + hi lo + lo hi -- three matrix instructions where the fp32 ones, at a sixteenth of the rate,
// would take the time of sixteen -- summed in 32 bits; lo lo is at most 2^-22 of the product, of
// either sign.  The floor under lo is 2^-25 of the scaled value: with e = 14, 2^-39, which rows far smaller than the others
// come to feel (at 1e-5 of them 2e-6 of themselves, at 1e-7 2e-4, after 5 steps; the whole stays at 1.3e-6, plain fp32 at 1.7e-6).
// b is kept without c0 I, and in the first step and while four or more follow x is carried in fp32 beside its
// pairs: early steps are little more than x = c0 x, and what is lost of a small singular value there
// is enlarged by every later step (final error on a 1024 x 1024 gradient: 4.2e-7 carried to the end,
// 5.2e-7 so, 7.8e-7 never; fp32 products give 1.3e-6).
//
// a and a a are symmetric: only tiles on and above the diagonal are computed and written twice.
//
// Operand form.  Every product here is P . Q^T with both operands read along k, so a matrix is kept
// as blocks of 16 rows x 32 columns, [column block][row block][hi, lo], and a block is the 1 KB that
// the 64 lanes of v_mfma_f32_16x16x32_f16 take as an operand, 16 bytes a lane: row lane & 15,
// columns 8 (lane >> 4) + 0..7.  A stage of a tile is one run of memory per operand, and LDS is
// written and read in lane order, without bank conflicts.  Rows and columns are padded with zeros
// to multiples of 32; x is kept along its columns and, for the product b x, along its rows.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "kernels.hpp"
#include "low_bits.hpp"

namespace cake {

namespace {

constexpr int BLOCK = 512;        // halves of one part of a 16 x 32 block
enum { NORM_CHUNKS = 512, MAX_SLICES = 32 };

// Element (row, col) of a matrix of row_blocks blocks of 16 rows: halves from its start to the hi part;
// the lo part is BLOCK further.
__device__ __forceinline__ size_t pair_at(int row, int col, int row_blocks)
{
    return ((size_t)(col >> 5) * row_blocks + (row >> 4)) * (2 * BLOCK) + ((row & 15) + ((col >> 3) & 3) * 16) * 8 + (col & 7);
}

// The same for the first element of the 16 x 16 half of a block at blocks (bi, bj) of 16, the same for a whole wave;
// behind it lies (row, col) at col / 8 * 128 + row * 8 + col % 8.
__device__ __forceinline__ size_t half_at(int bi, int bj, int row_blocks)
{
    return ((size_t)(bj >> 1) * row_blocks + bi) * (2 * BLOCK) + (bj & 1) * (BLOCK / 2);
}
// Where a lane finds rows 4 (lane >> 4) + 0..3 of column lane & 15 of a half that is kept turned: 4 consecutive halves
__device__ __forceinline__ unsigned turned_lane(unsigned lane) { return (lane >> 5) * 128 + (lane & 15) * 8 + (lane >> 4 & 1) * 4; }

// The carried x: blocks of 16 x 16 floats, four a lane as a product's results come out of the matrix pipe.
__device__ __forceinline__ size_t carried_at(int bi, int bj, int row_blocks) { return ((size_t)bj * row_blocks + bi) * 256; }

__device__ __forceinline__ void split(float v, _Float16& hi, _Float16& lo)
{
    hi = (_Float16)v;
    lo = (_Float16)(v - (float)hi);
}

// Sums of squares in 64 bits, so that no gradient is too small or too large for its norm.  Eight values a
// lane and load; the hardware takes them at any address.
template <int TYPE>
__global__ __launch_bounds__(256) void norm_partial_kernel(const typename Element<TYPE>::T* __restrict__ g, double* __restrict__ partial, size_t values)
{
    typedef typename Element<TYPE>::T T;
    __shared__ double red[4];
    g += (size_t)blockIdx.y * values;
    double sum = 0;
    const size_t step = (size_t)gridDim.x * 256 * 8;
    size_t i = ((size_t)blockIdx.x * 256 + threadIdx.x) * 8;
    for (; i + 8 <= values; i += step) {
        T v[8];
        __builtin_memcpy(v, g + i, sizeof v);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum += (double)(float)v[e] * (double)(float)v[e];
    }
    for (int e = 0; e < 8; ++e)   // the last, incomplete eight are one lane's
        if (i + e < values) sum += (double)(float)g[i + e] * (double)(float)g[i + e];
    for (int s = 32; s; s >>= 1) sum += __shfl_xor(sum, s);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) partial[blockIdx.y * NORM_CHUNKS + blockIdx.x] = red[0] + red[1] + red[2] + red[3];
}

// x0 = g / (norm + eps) in both orders.  m <= n are x's sides; `tall`: g is n x m.  A workgroup takes
// 64 x 64 of x through LDS, so that g is read and the blocks are written in whole lines.
__global__ __launch_bounds__(256) void normalize_kernel(const void* __restrict__ g, int type, const double* __restrict__ partial, int chunks,
                                                        double eps, float up, _Float16* __restrict__ x, _Float16* __restrict__ xt,
                                                        float* __restrict__ carried, int m, int n, int mb, int nb, bool tall, size_t x_stride)
{
    __shared__ float tile[64][65];
    __shared__ double red[4];
    const int tid = threadIdx.x, lane = tid & 63;
    const size_t base = (size_t)blockIdx.z * m * n;
    double sum = 0;
    for (int i = tid; i < chunks; i += 256) sum += partial[blockIdx.z * NORM_CHUNKS + i];
    for (int s = 32; s; s >>= 1) sum += __shfl_xor(sum, s);
    if (lane == 0) red[tid >> 6] = sum;
    __syncthreads();
    const double length = sqrt(red[0] + red[1] + red[2] + red[3]) + eps;
    const double by = length == 0 ? 0 : 1.0 / length;   // zeros stay zeros also without an eps
    const int i0 = blockIdx.y * 64, j0 = blockIdx.x * 64;   // of x
    for (int r = tid >> 6; r < 64; r += 4) {
        const int i = tall ? i0 + lane : i0 + r, j = tall ? j0 + r : j0 + lane;
        float v = 0;
        if (i < m && j < n) v = (float)((double)load_as_float(g, base + (tall ? (size_t)j * m + i : (size_t)i * n + j), type) * by);
        tile[i - i0][j - j0] = v;
    }
    __syncthreads();
    x += blockIdx.z * x_stride;
    xt += blockIdx.z * x_stride;
    carried += blockIdx.z * (x_stride / 2);
    for (int u = tid >> 6; u < 16; u += 4) {
        const int bi = i0 / 16 + (u >> 2), bj = j0 / 16 + (u & 3);
        if (bi >= mb || bj >= nb) continue;
        const int row = (u >> 2) * 16 + (lane >> 4) * 4, col = (u & 3) * 16 + (lane & 15);
        *reinterpret_cast<floatx4*>(carried + carried_at(bi, bj, mb) + lane * 4) =
            floatx4{tile[row][col], tile[row + 1][col], tile[row + 2][col], tile[row + 3][col]};
    }
    // 4 row blocks x 2 column blocks of x, and as many of its transpose
    for (int u = tid >> 6; u < 16; u += 4) {
        const bool turned = u >= 8;
        const int rb = (u & 7) >> 1, cb = u & 1;
        const int row = rb * 16 + (lane & 15), col = cb * 32 + (lane >> 4) * 8;
        f16x8 hi, lo;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            _Float16 h, l;
            split((turned ? tile[col + e][row] : tile[row][col + e]) * up, h, l);
            hi[e] = h;
            lo[e] = l;
        }
        const int row0 = (turned ? j0 : i0) + rb * 16, col0 = (turned ? i0 : j0) + cb * 32;
        const int row_blocks = turned ? nb : mb, col_blocks = (turned ? mb : nb) / 2;
        if (row0 / 16 >= row_blocks || col0 / 32 >= col_blocks) continue;
        _Float16* to = (turned ? xt : x) + pair_at(row0, col0, row_blocks) + lane * 8;
        *reinterpret_cast<f16x8*>(to) = hi;
        *reinterpret_cast<f16x8*>(to + BLOCK) = lo;
    }
}

enum { GRAM = 0, POLYNOMIAL = 1, APPLY = 2, FINISH = 3 };   // FINISH: the last step's APPLY, into the caller's matrix

struct PairGemm {
    const _Float16* p;        // rows i
    const _Float16* q;        // rows j
    const _Float16* a;        // POLYNOMIAL: a itself
    float* carried;           // APPLY, FINISH: x in fp32
    const _Float16* was_t;    // and the pairs of its transpose
    bool from_carried, to_carried;
    _Float16* out;            // GRAM, POLYNOMIAL: the symmetric result; APPLY: x
    _Float16* out_t;          // APPLY: its transpose
    void* result;             // FINISH
    float* partial;           // sums of K slices, or nullptr
    int type;                 // of the result
    bool tall;
    int mi, mj;               // the result's real sides
    int ib, jb, kb;           // blocks of 16 rows of either operand, of 32 columns
    int tiles_i, tiles_j, tiles;
    int slices;               // workgroups along k of a tile
    size_t p_stride, q_stride, a_stride, out_stride, result_stride;   // from one matrix of the batch to the next
    float unscale;            // of the accumulated product
    float c0, c1, c2;
    float a_unscale, up;      // of the parts of a or of x; 2^e of the result
};

// Tile number -> (ti, tj): all of them, ti fastest (workgroups that run together share columns of x),
// or of a symmetric result those with ti <= tj, column by column.
template <int MODE>
__device__ __forceinline__ void tile_of(int id, int tiles_i, int& ti, int& tj)
{
    if (MODE >= APPLY) {
        ti = id % tiles_i;
        tj = id / tiles_i;
    } else {
        tj = (int)((__builtin_sqrtf(8.f * id + 1.f) - 1.f) * 0.5f);
        while (tj * (tj + 1) / 2 > id) --tj;
        while ((tj + 1) * (tj + 2) / 2 <= id) ++tj;
        ti = id - tj * (tj + 1) / 2;
    }
}

// Workgroups are dealt out to the eight dies in turn, each with an L2 of its own.  Where k is sliced they are
// numbered so that a die's are consecutive and it reads an eighth of the operands, not all of them (a of 1024 x 4096
// in 7 slices 22 to 20 us); without slices either order takes the same time.
__device__ __forceinline__ int die_order(int id, int all)
{
    const int die = id & 7, each = all >> 3;
    return die * each + min(die, all & 7) + (id >> 3);
}

// a of the lanes where `upper` is not set and b of the lanes where it is, exchanged for the partner's other one
template <int PARTNER>
__device__ __forceinline__ void swap_across(unsigned& a, unsigned& b, bool upper)
{
    const unsigned got = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(upper ? a : b), PARTNER, 0xF, 0xF, true);
    a = upper ? got : a;
    b = upper ? b : got;
}

// Four values of one column (rows 4 (lane >> 4) + 0..3, column lane & 15 of block bi, bj) as pairs at
// [column][rows]: 8 bytes a lane and whole lines a wave.
__device__ __forceinline__ void store_along(_Float16* out, int bi, int bj, int row_blocks, f16x4 hi, f16x4 lo, int lane)
{
    _Float16* to = out + half_at(bj, bi, row_blocks) + turned_lane(lane);
    *reinterpret_cast<f16x4*>(to) = hi;
    *reinterpret_cast<f16x4*>(to + BLOCK) = lo;
}

// The same values at [row][columns]: four rows of a column to four columns of a row is a 4 x 4
// transposition among four lanes in a row, hi and lo in one word, so that the stores are 8 bytes a lane
// here too.
__device__ __forceinline__ void store_across(_Float16* out, int bi, int bj, int row_blocks, f16x4 hi, f16x4 lo, int lane)
{
    unsigned w[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const f16x2 both = {hi[r], lo[r]};
        w[r] = __builtin_bit_cast(unsigned, both);
    }
    swap_across<0xB1>(w[0], w[1], lane & 1);   // lane ^ 1
    swap_across<0xB1>(w[2], w[3], lane & 1);
    swap_across<0x4E>(w[0], w[2], lane & 2);   // lane ^ 2
    swap_across<0x4E>(w[1], w[3], lane & 2);
    uintx2 h, l;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        h[r] = (w[2 * r] & 0xFFFFu) | w[2 * r + 1] << 16;
        l[r] = w[2 * r] >> 16 | (w[2 * r + 1] & 0xFFFF0000u);
    }
    _Float16* to = out + half_at(bi, bj, row_blocks) + ((unsigned)(lane >> 3 & 1) * 128 + ((lane >> 4) * 4 + (lane & 3)) * 8 + (lane & 4));
    *reinterpret_cast<uintx2*>(to) = h;
    *reinterpret_cast<uintx2*>(to + BLOCK) = l;
}

__device__ __forceinline__ void split4(floatx4 v, float up, f16x4& hi, f16x4& lo)
{
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        _Float16 h, l;
        split(v[r] * up, h, l);
        hi[r] = h;
        lo[r] = l;
    }
}

// What becomes of one block of 16 x 16 sums: a lane holds column lane & 15 in four consecutive rows.
template <int MODE>
__device__ __forceinline__ void finish_block(const PairGemm& g, int z, int bi, int bj, bool mirror, floatx4 v, int lane)
{
    const int row = bi * 16 + (lane >> 4) * 4, c = bj * 16 + (lane & 15);
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] *= g.unscale;
    const size_t turned = half_at(bj, bi, g.jb) + turned_lane(lane);
    if (MODE >= APPLY) {
        floatx4* x = reinterpret_cast<floatx4*>(g.carried + z * (g.out_stride / 2) + carried_at(bi, bj, g.ib) + lane * 4);
        floatx4 was;
        if (g.from_carried) {
            was = *x;
        } else {
            const _Float16* t = g.was_t + z * g.out_stride + turned;
            const f16x4 h = *reinterpret_cast<const f16x4*>(t), l = *reinterpret_cast<const f16x4*>(t + BLOCK);
#pragma unroll
            for (int r = 0; r < 4; ++r) was[r] = ((float)h[r] + (float)l[r]) * g.a_unscale;
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = __builtin_fmaf(g.c0, was[r], v[r]);
        if (MODE == APPLY && g.to_carried) *x = v;
    }
    if (MODE == FINISH) {
        const size_t base = z * g.result_stride;
        if (c < g.mj) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (row + r < g.mi)
                    store_from_float(g.result, base + (g.tall ? (size_t)c * g.mi + row + r : (size_t)(row + r) * g.mj + c), g.type, v[r]);
        }
        return;
    }
    if (MODE == POLYNOMIAL) {
        const _Float16* a = g.a + z * g.a_stride + turned;
        const f16x4 ah = *reinterpret_cast<const f16x4*>(a), al = *reinterpret_cast<const f16x4*>(a + BLOCK);
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = g.c2 * v[r] + g.c1 * (((float)ah[r] + (float)al[r]) * g.a_unscale);
    }
    f16x4 hi, lo;
    split4(v, g.up, hi, lo);
    _Float16* out = g.out + z * g.out_stride;
    store_along(MODE == APPLY ? g.out_t + z * g.out_stride : out, bi, bj, g.jb, hi, lo, lane);
    // and in the other order: x itself, or the mirrored tile of a symmetric result
    if (MODE == APPLY || mirror) store_across(out, bi, bj, g.ib, hi, lo, lane);
}

// out = P . Q^T over WI x WJ waves of TI x TJ blocks of 16 x 16 each.  A stage is one column block (32
// of k) of both operands; the next one travels to registers while this one is multiplied and is
// written to the other half of LDS behind it.
template <int MODE, int WI, int WJ, int TI, int TJ>
__global__ __launch_bounds__(64 * WI * WJ) void pair_gemm_kernel(PairGemm g)
{
    constexpr int BI = WI * TI, BJ = WJ * TJ;                  // blocks per tile
    constexpr int STAGE = (BI + BJ) * 2 * BLOCK;               // halves
    constexpr int WAVES = WI * WJ;
    constexpr int LOADS = (BI + BJ) * 2 / WAVES;               // parts of 1 KB per wave
    constexpr int P_LOADS = BI * 2 / WAVES;
    static_assert(BI * 2 % WAVES == 0 && BJ * 2 % WAVES == 0, "either operand's parts must divide among the waves");
    extern __shared__ __align__(16) _Float16 stage[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wi = wave / WJ, wj = wave % WJ;

    int ti, tj;
    const int id = g.slices > 1 ? die_order(blockIdx.x, gridDim.x) : (int)blockIdx.x;
    const int slice = id / g.tiles, tile = id - slice * g.tiles;
    tile_of<MODE>(tile, g.tiles_i, ti, tj);
    const int k0 = (int)((long long)g.kb * slice / g.slices), k1 = (int)((long long)g.kb * (slice + 1) / g.slices);
    const _Float16* p = g.p + blockIdx.z * g.p_stride;
    const _Float16* q = g.q + blockIdx.z * g.q_stride;

    // the parts this wave fetches: block t of the tile (P's, then Q's), hi or lo; rows past the
    // operand's last block repeat that block, and their results are not stored
    const char* from_p = reinterpret_cast<const char*>(p);     // the same for every lane: addresses are scalars
    const char* from_q = reinterpret_cast<const char*>(q);
    const size_t step_p = (size_t)g.ib * 4 * BLOCK, step_q = (size_t)g.jb * 4 * BLOCK;
    from_p += k0 * step_p + (size_t)ti * BI * 4 * BLOCK;
    from_q += k0 * step_q + (size_t)tj * BJ * 4 * BLOCK;
    unsigned at_part[LOADS];   // within the tile: 32 bits, however long the side
#pragma unroll
    for (int l = 0; l < LOADS; ++l) {
        const int part = l * WAVES + wave, t = part >> 1;
        const int block = l < P_LOADS ? min(t, g.ib - 1 - ti * BI) : min(t - BI, g.jb - 1 - tj * BJ);
        at_part[l] = (unsigned)block * 4 * BLOCK + (part & 1) * 2 * BLOCK + lane * 16;
    }
    f16x8 next[LOADS];
    auto fetch = [&](int l) { next[l] = *reinterpret_cast<const f16x8*>((l < P_LOADS ? from_p : from_q) + at_part[l]); };
    auto put = [&](int l, int half) {
        *reinterpret_cast<f16x8*>(stage + half * STAGE + (l * WAVES + wave) * BLOCK + lane * 8) = next[l];
    };
    // to the column block `of`; past the last one the last is fetched again, and nobody reads it
    auto advance = [&](int of) {
        from_p += of < k1 ? step_p : 0;
        from_q += of < k1 ? step_q : 0;
    };

    floatx4 acc[TI][TJ];
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int j = 0; j < TJ; ++j) acc[i][j] = floatx4{0, 0, 0, 0};
#pragma unroll
    for (int l = 0; l < LOADS; ++l) fetch(l);
#pragma unroll
    for (int l = 0; l < LOADS; ++l) put(l, 0);
    advance(k0 + 1);
#pragma unroll
    for (int l = 0; l < LOADS; ++l) fetch(l);
    __syncthreads();
    for (int k = k0; k < k1; ++k) {
        const int half = (k - k0) & 1;
        const _Float16* at = stage + half * STAGE + lane * 8;
        const _Float16* at_p = at + wi * TI * 2 * BLOCK;
        const _Float16* at_q = at + (BI + wj * TJ) * 2 * BLOCK;
        advance(k + 2);
        f16x8 qh[TJ], ql[TJ], ph[2], pl[2];
#pragma unroll
        for (int j = 0; j < TJ; ++j) {
            qh[j] = *reinterpret_cast<const f16x8*>(at_q + j * 2 * BLOCK);
            ql[j] = *reinterpret_cast<const f16x8*>(at_q + j * 2 * BLOCK + BLOCK);
        }
        ph[0] = *reinterpret_cast<const f16x8*>(at_p);
        pl[0] = *reinterpret_cast<const f16x8*>(at_p + BLOCK);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < TI; ++i) {
            const int now = i & 1;
            if (i + 1 < TI) {
                ph[now ^ 1] = *reinterpret_cast<const f16x8*>(at_p + (i + 1) * 2 * BLOCK);
                pl[now ^ 1] = *reinterpret_cast<const f16x8*>(at_p + (i + 1) * 2 * BLOCK + BLOCK);
            }
            // this row of blocks' share of the next stage: out of the registers, and the stage after it in
#pragma unroll
            for (int l = i * LOADS / TI; l < (i + 1) * LOADS / TI; ++l) {
                put(l, half ^ 1);
                fetch(l);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < TJ; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pl[now], qh[j], acc[i][j], 0, 0, 0);
#pragma unroll
            for (int j = 0; j < TJ; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph[now], ql[j], acc[i][j], 0, 0, 0);
#pragma unroll
            for (int j = 0; j < TJ; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph[now], qh[j], acc[i][j], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
        __syncthreads();
    }

    if (g.partial) {
        float* to = g.partial + (((size_t)blockIdx.z * gridDim.x + id) * (BI * BJ)) * 256 + lane * 4;
#pragma unroll
        for (int i = 0; i < TI; ++i)
#pragma unroll
            for (int j = 0; j < TJ; ++j) *reinterpret_cast<floatx4*>(to + ((wi * TI + i) * BJ + wj * TJ + j) * 256) = acc[i][j];
        return;
    }
#pragma unroll
    for (int i = 0; i < TI; ++i) {
        const int bi = ti * BI + wi * TI + i;
#pragma unroll
        for (int j = 0; j < TJ; ++j) {
            const int bj = tj * BJ + wj * TJ + j;
            if (bi < g.ib && bj < g.jb) finish_block<MODE>(g, blockIdx.z, bi, bj, ti != tj, acc[i][j], lane);
        }
    }
}

// The K slices of every tile added up in order, a wave per block.
template <int MODE>
__global__ __launch_bounds__(256) void join_slices_kernel(PairGemm g, int tile_blocks)
{
    const int lane = threadIdx.x & 63;
    const int per_tile = tile_blocks * tile_blocks;
    const int unit = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tile = unit / per_tile, block = unit - tile * per_tile;
    if (tile >= g.tiles) return;
    int ti, tj;
    tile_of<MODE>(tile, g.tiles_i, ti, tj);
    const int bi = ti * tile_blocks + block / tile_blocks, bj = tj * tile_blocks + block % tile_blocks;
    if (bi >= g.ib || bj >= g.jb) return;
    const size_t step = (size_t)g.tiles * per_tile * 256;
    const float* from = g.partial + (size_t)blockIdx.z * g.slices * step + ((size_t)tile * per_tile + block) * 256 + lane * 4;
    floatx4 v = *reinterpret_cast<const floatx4*>(from);
    for (int s = 1; s < g.slices; ++s) v += *reinterpret_cast<const floatx4*>(from + s * step);
    finish_block<MODE>(g, blockIdx.z, bi, bj, ti != tj, v, lane);
}

// The four tiles, and what a stage of 32 columns and a tile's beginning and end take in microseconds
// (measured on sides of 256 to 4096): `alone` with one workgroup on a compute unit, `full`
// with as many as fit.
struct TileCost {
    int blocks, resident;
    float alone, full;
};
constexpr TileCost TILES[] = {{4, 4, 0.34f, 1.1f}, {8, 2, 0.75f, 1.42f}, {12, 1, 1.42f, 1.42f}, {16, 1, 2.35f, 2.35f}};
// The device's compute units; a number of this file, so that the size of the workspace and the order of
// the sums follow from the sizes alone.
constexpr int CUS = 256;
struct TileChoice {
    int which, slices;
};

int tile_count(int blocks, int ib, int jb, bool symmetric)
{
    const int i = (ib + blocks - 1) / blocks, j = (jb + blocks - 1) / blocks;
    return symmetric ? i * (i + 1) / 2 : i * j;
}

// The tile and the number of K slices with the least estimated time.  Slices give a result of few
// tiles to the whole device, at the price of a pass over the partial sums.
TileChoice choose_tile(int ib, int jb, int kb, bool symmetric, int batch)
{
    TileChoice best{0, 1};
    float least = 1e30f;
    for (int w = 0; w < 4; ++w) {
        const TileCost& t = TILES[w];
        const float tiles = (float)tile_count(t.blocks, ib, jb, symmetric) * batch;
        for (int s = 1; s <= MAX_SLICES && s <= kb; ++s) {
            const float groups = tiles * s;
            if (s > 1 && groups > CUS * t.resident) break;
            const float rounds = ceilf(groups / (CUS * t.resident));
            const float beside = fminf(ceilf(groups / CUS), (float)t.resident) - 1;   // others on the same compute unit
            const float stage = beside > 0 ? t.alone + (t.full - t.alone) * beside / (float)(t.resident - 1) : t.alone;
            float us = 3.f + rounds * (stage * ((kb + s - 1) / s) + 3.f);
            // partial sums out and back at about 6 TB/s, and a launch
            if (s > 1) us += 5.f + 0.15f * s + groups * t.blocks * t.blocks * 2048 / 6e6f;
            if (us < least) {
                least = us;
                best = {w, s};
            }
        }
    }
    return best;
}

template <int MODE, int WI, int WJ, int TI, int TJ>
hipError_t pair_gemm_on(PairGemm g, int batch, hipStream_t stream)
{
    static_assert(WI * TI == WJ * TJ, "square tiles");
    constexpr int BLOCKS = WI * TI;
    g.tiles_i = (g.ib + BLOCKS - 1) / BLOCKS;
    g.tiles_j = (g.jb + BLOCKS - 1) / BLOCKS;
    g.tiles = tile_count(BLOCKS, g.ib, g.jb, MODE < APPLY);
    constexpr size_t LDS = (size_t)2 * 2 * BLOCKS * 2 * BLOCK * sizeof(_Float16);
    auto kernel = &pair_gemm_kernel<MODE, WI, WJ, TI, TJ>;
    if (LDS > 64 * 1024) {
        hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)LDS);
        if (e != hipSuccess) return e;
    }
    kernel<<<dim3(g.tiles * g.slices, 1, batch), dim3(64 * WI * WJ), LDS, stream>>>(g);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || g.slices == 1) return e;
    join_slices_kernel<MODE><<<dim3((unsigned)((size_t)g.tiles * BLOCKS * BLOCKS + 3) / 4, 1, batch), 256, 0, stream>>>(g, BLOCKS);
    return hipGetLastError();
}

template <int MODE>
hipError_t pair_gemm(PairGemm g, int batch, float* partial, hipStream_t stream)
{
    const TileChoice t = choose_tile(g.ib, g.jb, g.kb, MODE < APPLY, batch);
    g.slices = t.slices;
    g.partial = t.slices > 1 ? partial : nullptr;
    switch (t.which) {
    case 0: return pair_gemm_on<MODE, 2, 2, 2, 2>(g, batch, stream);
    case 1: return pair_gemm_on<MODE, 2, 4, 4, 2>(g, batch, stream);
    case 2: return pair_gemm_on<MODE, 2, 4, 6, 3>(g, batch, stream);
    default: return pair_gemm_on<MODE, 2, 4, 8, 4>(g, batch, stream);
    }
}

// floats of partial sums that the choice above asks for
size_t slice_floats(int ib, int jb, int kb, bool symmetric, int batch)
{
    const TileChoice t = choose_tile(ib, jb, kb, symmetric, batch);
    if (t.slices == 1) return 0;
    const int blocks = TILES[t.which].blocks;
    return (size_t)tile_count(blocks, ib, jb, symmetric) * t.slices * batch * blocks * blocks * 256;
}

// ---- small matrices ------------------------------------------------------------------------
// One workgroup per matrix and one launch: a matrix whose pairs and whose square's pairs fit the LDS of a
// compute unit together (sides up to 128 x 160, 64 x 544, 32 x 1200).  x stays in registers in fp32, in
// blocks as they come out of the matrix pipe; its pairs are written to LDS along its columns for
// a = x x^T and then, over them, along its rows for b x.  Launches of a product each cost 5 to 6 us
// at these sizes whatever they do: 16 matrices of 96 x 130 took 98 us in 17 launches, 42 us in one.
// The products are bound by what LDS delivers, so a wave takes units of 2 x 2 blocks, half the operands a
// block, wherever there is more than a block or two for every wave.
enum { SMALL_WAVES = 16 };
constexpr int small_units(int x_side, int a_side) { return x_side == 2 && a_side == 1 ? 3 : 2; }   // of x in a wave; of the square it holds one

struct SmallArgs {
    const void* g;
    void* out;
    int type, m, n, mb, nb, steps;
    bool tall;
    float c0, c1, c2;
    double eps;
    float up_x, up_a, up_b;
};

// The sums over kb column blocks of a unit's products.  For a single block the next operands are on their way while
// these are multiplied, and the small products have a sum of their own, so that a matrix instruction
// waits for one before it rather than for two.
__device__ __forceinline__ void unit_product(const _Float16* p, const _Float16* q, int step_p, int step_q, int kb, floatx4 (&sum)[1][1])
{
    floatx4 acc = {0, 0, 0, 0}, low = {0, 0, 0, 0};
    f16x8 ph = *reinterpret_cast<const f16x8*>(p), pl = *reinterpret_cast<const f16x8*>(p + BLOCK);
    f16x8 qh = *reinterpret_cast<const f16x8*>(q), ql = *reinterpret_cast<const f16x8*>(q + BLOCK);
    for (int k = 1; k < kb; ++k) {
        p += step_p;
        q += step_q;
        const f16x8 nph = *reinterpret_cast<const f16x8*>(p), npl = *reinterpret_cast<const f16x8*>(p + BLOCK);
        const f16x8 nqh = *reinterpret_cast<const f16x8*>(q), nql = *reinterpret_cast<const f16x8*>(q + BLOCK);
        low = __builtin_amdgcn_mfma_f32_16x16x32_f16(pl, qh, low, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph, qh, acc, 0, 0, 0);
        low = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph, ql, low, 0, 0, 0);
        ph = nph;
        pl = npl;
        qh = nqh;
        ql = nql;
    }
    low = __builtin_amdgcn_mfma_f32_16x16x32_f16(pl, qh, low, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph, qh, acc, 0, 0, 0);
    low = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph, ql, low, 0, 0, 0);
    sum[0][0] = acc + low;
}
__device__ __forceinline__ void unit_product(const _Float16* p, const _Float16* q, int step_p, int step_q, int kb, floatx4 (&sum)[2][2])
{
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < 2; ++b) sum[a][b] = floatx4{0, 0, 0, 0};
    for (int k = 0; k < kb; ++k) {
        f16x8 ph[2], pl[2], qh[2], ql[2];
#pragma unroll
        for (int a = 0; a < 2; ++a) {
            ph[a] = *reinterpret_cast<const f16x8*>(p + a * 2 * BLOCK);
            pl[a] = *reinterpret_cast<const f16x8*>(p + a * 2 * BLOCK + BLOCK);
            qh[a] = *reinterpret_cast<const f16x8*>(q + a * 2 * BLOCK);
            ql[a] = *reinterpret_cast<const f16x8*>(q + a * 2 * BLOCK + BLOCK);
        }
        __builtin_amdgcn_sched_barrier(0);   // one wait for all eight, not one for each
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int b = 0; b < 2; ++b) sum[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pl[a], qh[b], sum[a][b], 0, 0, 0);
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int b = 0; b < 2; ++b) sum[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph[a], ql[b], sum[a][b], 0, 0, 0);
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int b = 0; b < 2; ++b) sum[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph[a], qh[b], sum[a][b], 0, 0, 0);
        p += step_p;
        q += step_q;
    }
}

// XS, AS: sides of a unit of x and of the square.
template <int XS, int AS>
__global__ __launch_bounds__(64 * SMALL_WAVES) void small_matrices_kernel(SmallArgs s)
{
    extern __shared__ __align__(16) _Float16 stage[];
    __shared__ double norms[SMALL_WAVES];
    constexpr int UNITS = small_units(XS, AS);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    _Float16* const xs = stage;                          // pairs of x, then of its transpose
    _Float16* const as = stage + s.mb * s.nb * BLOCK;    // pairs of a, then of b
    const int rows = s.mb / XS, units = rows * (s.nb / XS), squares = (s.mb / AS) * (s.mb / AS + 1) / 2;
    const size_t base = (size_t)blockIdx.x * s.m * s.n;
    auto index = [&](int i, int j) { return base + (s.tall ? (size_t)j * s.m + i : (size_t)i * s.n + j); };

    // this wave's blocks of x, and those of the square
    int x_bi[UNITS], x_bj[UNITS], a_bi, a_bj;
#pragma unroll
    for (int t = 0; t < UNITS; ++t) {
        x_bi[t] = (wave + t * waves) % rows * XS;
        x_bj[t] = (wave + t * waves) / rows * XS;
    }
    tile_of<GRAM>(wave, 0, a_bi, a_bj);
    a_bi *= AS;
    a_bj *= AS;

    floatx4 x[UNITS][XS][XS];
    double sum = 0;
#pragma unroll
    for (int t = 0; t < UNITS; ++t)
#pragma unroll
        for (int a = 0; a < XS; ++a)
#pragma unroll
            for (int b = 0; b < XS; ++b) {
                x[t][a][b] = floatx4{0, 0, 0, 0};
                if (wave + t * waves < units) {
                    const int i = (x_bi[t] + a) * 16 + (lane >> 4) * 4, j = (x_bj[t] + b) * 16 + (lane & 15);
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (i + r < s.m && j < s.n) {
                            const float v = load_as_float(s.g, index(i + r, j), s.type);
                            x[t][a][b][r] = v;
                            sum += (double)v * (double)v;
                        }
                }
            }
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    if (lane == 0) norms[wave] = sum;
    __syncthreads();
    sum = 0;
    for (int w = 0; w < waves; ++w) sum += norms[w];
    const double length = sqrt(sum) + s.eps;
    const double by = length == 0 ? 0 : 1.0 / length;   // zeros stay zeros also without an eps
#pragma unroll
    for (int t = 0; t < UNITS; ++t)
#pragma unroll
        for (int a = 0; a < XS; ++a)
#pragma unroll
            for (int b = 0; b < XS; ++b)
#pragma unroll
                for (int r = 0; r < 4; ++r) x[t][a][b][r] = (float)((double)x[t][a][b][r] * by);

    const float down_aa = 1.f / (s.up_a * s.up_a), down_xx = 1.f / (s.up_x * s.up_x), down_bx = 1.f / (s.up_b * s.up_x), down_a = 1.f / s.up_a;
    auto store_x = [&](bool along) {
#pragma unroll
        for (int t = 0; t < UNITS; ++t)
            if (wave + t * waves < units) {
#pragma unroll
                for (int a = 0; a < XS; ++a)
#pragma unroll
                    for (int b = 0; b < XS; ++b) {
                        f16x4 hi, lo;
                        split4(x[t][a][b], s.up_x, hi, lo);
                        if (along) store_along(xs, x_bi[t] + a, x_bj[t] + b, s.nb, hi, lo, lane);
                        else store_across(xs, x_bi[t] + a, x_bj[t] + b, s.mb, hi, lo, lane);
                    }
            }
    };
    const int step_a = s.mb * 2 * BLOCK;
    for (int step = 0; step < s.steps; ++step) {
        store_x(false);
        __syncthreads();
        floatx4 square[AS][AS];
        auto store_squares = [&](float up) {
            if (wave < squares) {
#pragma unroll
                for (int a = 0; a < AS; ++a)
#pragma unroll
                    for (int b = 0; b < AS; ++b) {
                        const int bi = a_bi + a, bj = a_bj + b;
                        if (bi > bj) continue;   // the lower half of a unit on the diagonal comes from its upper one
                        f16x4 hi, lo;
                        split4(square[a][b], up, hi, lo);
                        store_along(as, bi, bj, s.mb, hi, lo, lane);
                        if (bi != bj) store_across(as, bi, bj, s.mb, hi, lo, lane);
                    }
            }
        };
        if (wave < squares) {
            unit_product(xs + a_bi * 2 * BLOCK + lane * 8, xs + a_bj * 2 * BLOCK + lane * 8, step_a, step_a, s.nb / 2, square);
#pragma unroll
            for (int a = 0; a < AS; ++a)
#pragma unroll
                for (int b = 0; b < AS; ++b)
#pragma unroll
                    for (int r = 0; r < 4; ++r) square[a][b][r] *= down_xx;
        }
        store_squares(s.up_a);   // the first time into memory that nobody reads, then behind the barrier after b x
        __syncthreads();
        store_x(true);           // a is complete: nobody reads x along its columns any more
        if (wave < squares) {
            unit_product(as + a_bi * 2 * BLOCK + lane * 8, as + a_bj * 2 * BLOCK + lane * 8, step_a, step_a, s.mb / 2, square);
#pragma unroll
            for (int a = 0; a < AS; ++a)
#pragma unroll
                for (int b = 0; b < AS; ++b) {
                    const _Float16* at = as + half_at(a_bj + b, a_bi + a, s.mb) + turned_lane(lane);
                    const f16x4 ah = *reinterpret_cast<const f16x4*>(at), al = *reinterpret_cast<const f16x4*>(at + BLOCK);
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        square[a][b][r] = s.c2 * (square[a][b][r] * down_aa) + s.c1 * (((float)ah[r] + (float)al[r]) * down_a);
                }
        }
        __syncthreads();
        store_squares(s.up_b);
        __syncthreads();
#pragma unroll
        for (int t = 0; t < UNITS; ++t)
            if (wave + t * waves < units) {
                floatx4 v[XS][XS];
                unit_product(as + x_bi[t] * 2 * BLOCK + lane * 8, xs + x_bj[t] * 2 * BLOCK + lane * 8, step_a, s.nb * 2 * BLOCK, s.mb / 2, v);
#pragma unroll
                for (int a = 0; a < XS; ++a)
#pragma unroll
                    for (int b = 0; b < XS; ++b)
#pragma unroll
                        for (int r = 0; r < 4; ++r) x[t][a][b][r] = __builtin_fmaf(s.c0, x[t][a][b][r], v[a][b][r] * down_bx);
            }
        __syncthreads();
    }
#pragma unroll
    for (int t = 0; t < UNITS; ++t)
        if (wave + t * waves < units) {
#pragma unroll
            for (int a = 0; a < XS; ++a)
#pragma unroll
                for (int b = 0; b < XS; ++b) {
                    const int i = (x_bi[t] + a) * 16 + (lane >> 4) * 4, j = (x_bj[t] + b) * 16 + (lane & 15);
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (i + r < s.m && j < s.n) store_from_float(s.out, index(i + r, j), s.type, x[t][a][b][r]);
                }
        }
}

// Sides of the units: single blocks where they are no more than two a wave (the square: one).
int small_x_side(int mb, int nb) { return mb * nb <= 2 * SMALL_WAVES ? 1 : 2; }
int small_a_side(int mb) { return mb <= 4 ? 1 : 2; }
int small_x_units(int mb, int nb) { return mb * nb / (small_x_side(mb, nb) * small_x_side(mb, nb)); }
int small_a_units(int mb)
{
    const int side = mb / small_a_side(mb);
    return side * (side + 1) / 2;
}

// a block of 16 x 32 pairs is 2 KB: mb nb / 2 of them for x, mb mb / 2 for the square, 1 KB left for the norm
bool small_fits(int mb, int nb)
{
    return mb * nb + mb * mb <= 159 && small_x_units(mb, nb) <= SMALL_WAVES * small_units(small_x_side(mb, nb), small_a_side(mb)) && small_a_units(mb) <= SMALL_WAVES;
}

}  // namespace

namespace {

struct OrthogonalizeLayout {      // of one pass; offsets are bytes into the workspace
    int m, n;                     // the shorter and the longer side
    int mb, nb;                   // in blocks of 16, even
    size_t x_halves, a_halves;    // of one matrix of the batch; the carried x has x_halves / 2 floats
    size_t x, xt0, xt1, a, b, partial, carried, slices, bytes;
};

OrthogonalizeLayout layout_of(int batch, int rows, int cols)
{
    OrthogonalizeLayout l;
    l.m = rows < cols ? rows : cols;
    l.n = rows < cols ? cols : rows;
    l.mb = (l.m + 31) / 32 * 2;
    l.nb = (l.n + 31) / 32 * 2;
    l.x_halves = (size_t)l.mb * l.nb * BLOCK;        // blocks of 16 x 32, two parts each
    l.a_halves = (size_t)l.mb * l.mb * BLOCK;
    l.x = 0;
    l.xt0 = l.x + (size_t)batch * l.x_halves * 2;
    l.xt1 = l.xt0 + (size_t)batch * l.x_halves * 2;
    l.a = l.xt1 + (size_t)batch * l.x_halves * 2;
    l.b = l.a + (size_t)batch * l.a_halves * 2;
    l.partial = l.b + (size_t)batch * l.a_halves * 2;
    l.carried = l.partial + (size_t)batch * NORM_CHUNKS * sizeof(double);
    l.slices = l.carried + (size_t)batch * l.x_halves * 2;
    const size_t floats[3] = {slice_floats(l.mb, l.mb, l.nb / 2, true, batch), slice_floats(l.mb, l.mb, l.mb / 2, true, batch),
                              slice_floats(l.mb, l.nb, l.mb / 2, false, batch)};
    l.bytes = small_fits(l.mb, l.nb) ? 0 : l.slices + std::max(floats[0], std::max(floats[1], floats[2])) * sizeof(float);
    return l;
}

// Matrices beyond PASS_VALUES together are taken some at a time, as evenly as they divide: the workspace holds 16 to
// 24 bytes a value, and a device that is full gains nothing from more (8 of 4096 x 4096 take 28.2 ms, 8 times one of them; 16
// of 1024 x 4096, which one pass takes, 4.2 ms, 16 of them by themselves 6.5).
constexpr size_t PASS_VALUES = (size_t)1 << 26;

int passes_of(int batch, int rows, int cols)
{
    const OrthogonalizeLayout one = layout_of(1, rows, cols);
    if (small_fits(one.mb, one.nb)) return 1;
    const size_t values = (size_t)one.mb * one.nb * 256;
    const size_t most = values < PASS_VALUES ? PASS_VALUES / values : 1;
    return (int)((batch + most - 1) / most);
}

hipError_t launch_pass(const void* g, void* out, int type, int batch, int rows, int cols, int steps, double c0, double c1, double c2, double eps,
                       const OrthogonalizeScales& sc, void* workspace, hipStream_t stream);

}  // namespace

size_t orthogonalize_workspace(int batch, int rows, int cols)
{
    const int passes = passes_of(batch, rows, cols);
    // a pass of one matrix less may ask for more slices
    return std::max(layout_of(batch / passes, rows, cols).bytes, layout_of((batch + passes - 1) / passes, rows, cols).bytes);
}

hipError_t launch_orthogonalize(const void* g, void* out, int type, int batch, int rows, int cols, int steps, double c0, double c1,
                                double c2, double eps, const OrthogonalizeScales& sc, void* workspace, hipStream_t stream)
{
    const int passes = passes_of(batch, rows, cols);
    const size_t bytes = (size_t)rows * cols * type_bytes(type);
    for (int p = 0; p < passes; ++p) {
        const int from = (int)((long long)batch * p / passes), to = (int)((long long)batch * (p + 1) / passes);
        const hipError_t e = launch_pass(static_cast<const char*>(g) + from * bytes, static_cast<char*>(out) + from * bytes, type, to - from, rows, cols,
                                         steps, c0, c1, c2, eps, sc, workspace, stream);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

namespace {

hipError_t launch_pass(const void* g, void* out, int type, int batch, int rows, int cols, int steps, double c0, double c1, double c2, double eps,
                       const OrthogonalizeScales& sc, void* workspace, hipStream_t stream)
{
    const OrthogonalizeLayout l = layout_of(batch, rows, cols);
    const float up_x = ldexpf(1.f, sc.ex), up_a = ldexpf(1.f, sc.ea), up_b = ldexpf(1.f, sc.eb);
    const bool tall = rows > cols;
    if (small_fits(l.mb, l.nb)) {
        SmallArgs a{g, out, type, l.m, l.n, l.mb, l.nb, steps, tall, (float)c0, (float)c1, (float)c2, eps, up_x, up_a, up_b};
        const size_t lds = (size_t)(l.mb * l.nb + l.mb * l.mb) * 1024;
        const int waves = std::min<int>(SMALL_WAVES, std::max(small_x_units(l.mb, l.nb), small_a_units(l.mb)));
        auto kernel = small_a_side(l.mb) == 2 ? &small_matrices_kernel<2, 2>
                                              : small_x_side(l.mb, l.nb) == 2 ? &small_matrices_kernel<2, 1> : &small_matrices_kernel<1, 1>;
        if (lds > 63 * 1024) {
            hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
            if (e != hipSuccess) return e;
        }
        kernel<<<batch, 64 * waves, lds, stream>>>(a);
        return hipGetLastError();
    }
    char* ws = static_cast<char*>(workspace);
    _Float16* x = reinterpret_cast<_Float16*>(ws + l.x);
    _Float16* xt[2] = {reinterpret_cast<_Float16*>(ws + l.xt0), reinterpret_cast<_Float16*>(ws + l.xt1)};
    _Float16* a = reinterpret_cast<_Float16*>(ws + l.a);
    _Float16* b = reinterpret_cast<_Float16*>(ws + l.b);
    double* partial = reinterpret_cast<double*>(ws + l.partial);
    float* carried = reinterpret_cast<float*>(ws + l.carried);
    float* slices = reinterpret_cast<float*>(ws + l.slices);
    const size_t values = (size_t)l.m * l.n;
    const size_t want = (values + 8191) / 8192;
    const int chunks = want < NORM_CHUNKS ? (int)want : NORM_CHUNKS;
    const dim3 norm_grid(chunks, batch);
    if (type == CAKE_HIP_F32) norm_partial_kernel<CAKE_HIP_F32><<<norm_grid, 256, 0, stream>>>(static_cast<const float*>(g), partial, values);
    else if (type == CAKE_HIP_F16) norm_partial_kernel<CAKE_HIP_F16><<<norm_grid, 256, 0, stream>>>(static_cast<const _Float16*>(g), partial, values);
    else norm_partial_kernel<CAKE_HIP_BF16><<<norm_grid, 256, 0, stream>>>(static_cast<const __bf16*>(g), partial, values);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    normalize_kernel<<<dim3((l.nb + 3) / 4, (l.mb + 3) / 4, batch), 256, 0, stream>>>(g, type, partial, chunks, eps, up_x, x, xt[0], carried, l.m,
                                                                                     l.n, l.mb, l.nb, tall, l.x_halves);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    for (int s = 0; s < steps; ++s) {
        PairGemm k{};
        k.p = k.q = x;
        k.out = a;
        k.mi = k.mj = l.m;
        k.ib = k.jb = l.mb;
        k.kb = l.nb / 2;
        k.p_stride = k.q_stride = l.x_halves;
        k.out_stride = l.a_halves;
        k.unscale = 1.f / (up_x * up_x);
        k.up = up_a;
        if ((e = pair_gemm<GRAM>(k, batch, slices, stream)) != hipSuccess) return e;
        k.p = k.q = k.a = a;
        k.out = b;
        k.kb = l.mb / 2;
        k.p_stride = k.q_stride = k.a_stride = l.a_halves;
        k.unscale = 1.f / (up_a * up_a);
        k.a_unscale = 1.f / up_a;
        k.up = up_b;
        k.c0 = (float)c0;
        k.c1 = (float)c1;
        k.c2 = (float)c2;
        if ((e = pair_gemm<POLYNOMIAL>(k, batch, slices, stream)) != hipSuccess) return e;
        const bool last = s == steps - 1;
        k.p = b;
        k.q = xt[s & 1];
        k.carried = carried;
        k.was_t = xt[s & 1];
        // what an error in x grows to depends on the steps that follow: x in 32 bits while four or more do, and in the
        // first step, whose x lies there in 32 bits whatever follows
        k.from_carried = s == 0 || steps - s >= 4;
        k.to_carried = steps - s >= 5;
        k.a_unscale = 1.f / up_x;
        k.out = x;
        k.out_t = xt[(s & 1) ^ 1];
        k.result = out;
        k.type = type;
        k.tall = tall;
        k.mj = l.n;
        k.jb = l.nb;
        k.q_stride = k.out_stride = l.x_halves;
        k.result_stride = values;
        k.unscale = 1.f / (up_b * up_x);
        k.up = up_x;
        e = last ? pair_gemm<FINISH>(k, batch, slices, stream) : pair_gemm<APPLY>(k, batch, slices, stream);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace

}  // namespace cake
