// orthogonalize.hip -- Newton-Schulz iterations on a batch of matrices:
//   x = g / (|g|_F + eps), then steps times  a = x x^T,  b = c0 I + c1 a + c2 a a,  x = b x
// (for more rows than columns on the transpose).
//
// All products run on the 16-bit matrix pipe at 32-bit accuracy.  A value v is kept as two fp16
// numbers, hi = fp16(v 2^e) and lo = fp16(v 2^e - hi): 11 significant bits each and the sign of lo
// make 2^-24 of relative error, and the power of two e keeps both parts in fp16's range (the
// iteration's values are bounded by its coefficients, so e is known beforehand).  A product is then
// hi hi + hi lo + lo hi -- three matrix instructions where the fp32 ones, at a sixteenth of the rate,
// would take the time of sixteen -- summed in 32 bits; lo lo is below 2^-24 of the product.  The
// floor under lo is 2^-25 of the scaled value: with e = 14, 2^-39 of the largest a value can be.
//
// a, a a and b are symmetric: only tiles on and above the diagonal are computed and written twice.
//
// Operand form.  Every product here is P . Q^T with both operands read along k, so a matrix is kept
// as blocks of 16 rows x 32 columns, [column block][row block][hi, lo], and a block is the 1 KB that
// the 64 lanes of v_mfma_f32_16x16x32_f16 take as an operand, 16 bytes a lane: row lane & 15,
// columns 8 (lane >> 4) + 0..7.  A stage of a tile is one run of memory per operand, and LDS is
// written and read in lane order, without bank conflicts.  Rows and columns are padded with zeros
// to multiples of 32; x is kept along its columns and, for the product b x, along its rows.
#include <hip/hip_runtime.h>

#include "kernels.hpp"
#include "low_bits.hpp"

namespace cake {

namespace {

constexpr int BLOCK = 512;        // halves of one part of a 16 x 32 block
enum { NORM_CHUNKS = 512 };

// Element (row, col) of a matrix of row_blocks blocks of 16 rows: halves from its start to the hi part;
// the lo part is BLOCK further.
__device__ __forceinline__ size_t pair_at(int row, int col, int row_blocks)
{
    return ((size_t)(col >> 5) * row_blocks + (row >> 4)) * (2 * BLOCK) + ((row & 15) + ((col >> 3) & 3) * 16) * 8 + (col & 7);
}

__device__ __forceinline__ void split(float v, _Float16& hi, _Float16& lo)
{
    hi = (_Float16)v;
    lo = (_Float16)(v - (float)hi);
}

// Sums of squares in 64 bits, so that no gradient is too small or too large for its norm.
__global__ __launch_bounds__(256) void norm_partial_kernel(const void* __restrict__ g, int type, double* __restrict__ partial, size_t values)
{
    __shared__ double red[4];
    const size_t base = (size_t)blockIdx.y * values;
    double sum = 0;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < values; i += (size_t)gridDim.x * 256) {
        const double v = (double)load_as_float(g, base + i, type);
        sum += v * v;
    }
    for (int s = 32; s; s >>= 1) sum += __shfl_xor(sum, s);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) partial[blockIdx.y * NORM_CHUNKS + blockIdx.x] = red[0] + red[1] + red[2] + red[3];
}

// x0 = g / (norm + eps) in both orders.  m <= n are x's sides; `tall`: g is n x m.  A workgroup takes
// 64 x 64 of x through LDS, so that g is read and the blocks are written in whole lines.
__global__ __launch_bounds__(256) void normalize_kernel(const void* __restrict__ g, int type, const double* __restrict__ partial, int chunks,
                                                        double eps, float up, _Float16* __restrict__ x, _Float16* __restrict__ xt, int m,
                                                        int n, int mb, int nb, bool tall, size_t x_stride)
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
        if (i < m && j < n) v = (float)((double)load_as_float(g, base + (tall ? (size_t)j * m + i : (size_t)i * n + j), type) * by) * up;
        tile[i - i0][j - j0] = v;
    }
    __syncthreads();
    x += blockIdx.z * x_stride;
    xt += blockIdx.z * x_stride;
    // 4 row blocks x 2 column blocks of x, and as many of its transpose
    for (int u = tid >> 6; u < 16; u += 4) {
        const bool turned = u >= 8;
        const int rb = (u & 7) >> 1, cb = u & 1;
        const int row = rb * 16 + (lane & 15), col = cb * 32 + (lane >> 4) * 8;
        f16x8 hi, lo;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            _Float16 h, l;
            split(turned ? tile[col + e][row] : tile[row][col + e], h, l);
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

enum { GRAM = 0, POLYNOMIAL = 1, APPLY = 2 };

struct PairGemm {
    const _Float16* p;        // rows i
    const _Float16* q;        // rows j
    const _Float16* a;        // POLYNOMIAL: a itself
    _Float16* out;            // GRAM, POLYNOMIAL: the symmetric result; APPLY: x (or nullptr on the last step)
    _Float16* out_t;          // APPLY: its transpose
    void* result;             // APPLY, last step: the caller's matrix
    int type;                 // of the result
    bool tall;
    int mi, mj;               // the result's real sides
    int ib, jb, kb;           // blocks of 16 rows of either operand, of 32 columns
    int tiles_i, tiles_j;
    size_t p_stride, q_stride, a_stride, out_stride, result_stride;   // from one matrix of the batch to the next
    float unscale;            // of the accumulated product
    float c0, c1, c2;
    float a_unscale, up;      // of a's parts; 2^e of the result
};

// out = P . Q^T over WI x WJ waves of TI x TJ blocks of 16 x 16 each.  A stage is one column block (32
// of k) of both operands; the next one travels to registers while this one is multiplied and is
// written to the other half of LDS behind it.
template <int MODE, int WI, int WJ, int TI, int TJ>
__global__ __launch_bounds__(64 * WI * WJ) void pair_gemm_kernel(PairGemm g)
{
    constexpr int BI = WI * TI, BJ = WJ * TJ;                  // blocks per tile
    constexpr int STAGE = (BI + BJ) * 2 * BLOCK;               // halves
    constexpr int LOADS = (BI + BJ) * 2 / (WI * WJ);           // parts of 1 KB per wave
    static_assert((BI + BJ) * 2 % (WI * WJ) == 0, "parts must divide among the waves");
    extern __shared__ __align__(16) _Float16 stage[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wi = wave / WJ, wj = wave % WJ;

    int ti, tj;
    if (MODE == APPLY) {
        ti = blockIdx.x % g.tiles_i;
        tj = blockIdx.x / g.tiles_i;
    } else {   // tiles with ti <= tj, column by column
        const int id = blockIdx.x;
        tj = (int)((__builtin_sqrtf(8.f * id + 1.f) - 1.f) * 0.5f);
        while (tj * (tj + 1) / 2 > id) --tj;
        while ((tj + 1) * (tj + 2) / 2 <= id) ++tj;
        ti = id - tj * (tj + 1) / 2;
    }
    const _Float16* p = g.p + blockIdx.z * g.p_stride;
    const _Float16* q = g.q + blockIdx.z * g.q_stride;

    // the parts this wave fetches: block t of the tile (P's, then Q's), hi or lo; rows past the
    // operand's last block repeat that block, and their results are not stored
    const _Float16* from[LOADS];
    size_t step[LOADS];
#pragma unroll
    for (int l = 0; l < LOADS; ++l) {
        const int part = wave * LOADS + l, t = part >> 1;
        const bool of_p = t < BI;
        const int block = of_p ? min(ti * BI + t, g.ib - 1) : min(tj * BJ + t - BI, g.jb - 1);
        from[l] = (of_p ? p : q) + (size_t)block * 2 * BLOCK + (part & 1) * BLOCK + lane * 8;
        step[l] = (size_t)(of_p ? g.ib : g.jb) * 2 * BLOCK;
    }
    f16x8 next[LOADS];
    auto fetch = [&]() {
#pragma unroll
        for (int l = 0; l < LOADS; ++l) {
            next[l] = *reinterpret_cast<const f16x8*>(from[l]);
            from[l] += step[l];
        }
    };
    auto put = [&](int half) {
#pragma unroll
        for (int l = 0; l < LOADS; ++l)
            *reinterpret_cast<f16x8*>(stage + half * STAGE + (wave * LOADS + l) * BLOCK + lane * 8) = next[l];
    };

    floatx4 acc[TI][TJ];
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int j = 0; j < TJ; ++j) acc[i][j] = floatx4{0, 0, 0, 0};
    fetch();
    put(0);
    __syncthreads();
    for (int k = 0; k < g.kb; ++k) {
        if (k + 1 < g.kb) fetch();
        const _Float16* at = stage + (k & 1) * STAGE + lane * 8;
        const _Float16* at_p = at + wi * TI * 2 * BLOCK;
        const _Float16* at_q = at + (BI + wj * TJ) * 2 * BLOCK;
        f16x8 qh[TJ], ql[TJ];
#pragma unroll
        for (int j = 0; j < TJ; ++j) {
            qh[j] = *reinterpret_cast<const f16x8*>(at_q + j * 2 * BLOCK);
            ql[j] = *reinterpret_cast<const f16x8*>(at_q + j * 2 * BLOCK + BLOCK);
        }
#pragma unroll
        for (int i = 0; i < TI; ++i) {
            const f16x8 ph = *reinterpret_cast<const f16x8*>(at_p + i * 2 * BLOCK);
            const f16x8 pl = *reinterpret_cast<const f16x8*>(at_p + i * 2 * BLOCK + BLOCK);
#pragma unroll
            for (int j = 0; j < TJ; ++j) {
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pl, qh[j], acc[i][j], 0, 0, 0);
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph, ql[j], acc[i][j], 0, 0, 0);
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph, qh[j], acc[i][j], 0, 0, 0);
            }
        }
        if (k + 1 < g.kb) put((k + 1) & 1);
        __syncthreads();
    }

    // a lane holds column col of a block in four consecutive rows
    const int col = lane & 15, row4 = (lane >> 4) * 4;
    _Float16* out = g.out ? g.out + blockIdx.z * g.out_stride : nullptr;
#pragma unroll
    for (int i = 0; i < TI; ++i) {
        const int bi = ti * BI + wi * TI + i;
        if (bi >= g.ib) continue;
#pragma unroll
        for (int j = 0; j < TJ; ++j) {
            const int bj = tj * BJ + wj * TJ + j;
            if (bj >= g.jb) continue;
            const int row = bi * 16 + row4, c = bj * 16 + col;
            floatx4 v;
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] = acc[i][j][r] * g.unscale;
            if (MODE == APPLY && !out) {
                const size_t base = blockIdx.z * g.result_stride;
                if (c < g.mj) {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (row + r < g.mi)
                            store_from_float(g.result, base + (g.tall ? (size_t)c * g.mi + row + r : (size_t)(row + r) * g.mj + c), g.type, v[r]);
                }
                continue;
            }
            const size_t turned = pair_at(c, row, g.jb);   // (column, rows): 4 consecutive halves
            if (MODE == POLYNOMIAL) {
                const _Float16* a = g.a + blockIdx.z * g.a_stride + turned;
                const f16x4 ah = *reinterpret_cast<const f16x4*>(a), al = *reinterpret_cast<const f16x4*>(a + BLOCK);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float av = ((float)ah[r] + (float)al[r]) * g.a_unscale;
                    v[r] = g.c2 * v[r] + (g.c1 * av + (row + r == c ? g.c0 : 0.f));
                }
            }
            f16x4 hi, lo;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                _Float16 h, l;
                split(v[r] * g.up, h, l);
                hi[r] = h;
                lo[r] = l;
            }
            _Float16* to = (MODE == APPLY ? g.out_t + blockIdx.z * g.out_stride : out) + turned;
            *reinterpret_cast<f16x4*>(to) = hi;
            *reinterpret_cast<f16x4*>(to + BLOCK) = lo;
            // and in the other order: x itself, or the mirrored tile of a symmetric result
            if (MODE == APPLY || ti != tj) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    _Float16* also = out + pair_at(row + r, c, g.ib);
                    also[0] = hi[r];
                    also[BLOCK] = lo[r];
                }
            }
        }
    }
}

template <int MODE>
hipError_t pair_gemm(PairGemm g, int batch, hipStream_t stream)
{
    constexpr int W = 2, T = 4;
    g.tiles_i = (g.ib + W * T - 1) / (W * T);
    g.tiles_j = (g.jb + W * T - 1) / (W * T);
    const int tiles = MODE == APPLY ? g.tiles_i * g.tiles_j : g.tiles_i * (g.tiles_i + 1) / 2;
    const size_t lds = (size_t)2 * 2 * W * T * 2 * BLOCK * sizeof(_Float16);
    pair_gemm_kernel<MODE, W, W, T, T><<<dim3(tiles, 1, batch), dim3(64 * W * W), lds, stream>>>(g);
    return hipGetLastError();
}

}  // namespace

OrthogonalizeLayout orthogonalize_layout(int batch, int rows, int cols)
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
    l.bytes = l.partial + (size_t)batch * NORM_CHUNKS * sizeof(double);
    return l;
}

hipError_t launch_orthogonalize(const void* g, void* out, int type, int batch, int rows, int cols, int steps, double c0, double c1,
                                double c2, double eps, const OrthogonalizeScales& sc, void* workspace, hipStream_t stream)
{
    const OrthogonalizeLayout l = orthogonalize_layout(batch, rows, cols);
    char* ws = static_cast<char*>(workspace);
    _Float16* x = reinterpret_cast<_Float16*>(ws + l.x);
    _Float16* xt[2] = {reinterpret_cast<_Float16*>(ws + l.xt0), reinterpret_cast<_Float16*>(ws + l.xt1)};
    _Float16* a = reinterpret_cast<_Float16*>(ws + l.a);
    _Float16* b = reinterpret_cast<_Float16*>(ws + l.b);
    double* partial = reinterpret_cast<double*>(ws + l.partial);
    const size_t values = (size_t)l.m * l.n;
    const bool tall = rows > cols;
    const size_t want = (values + 8191) / 8192;
    const int chunks = want < NORM_CHUNKS ? (int)want : NORM_CHUNKS;
    norm_partial_kernel<<<dim3(chunks, batch), 256, 0, stream>>>(g, type, partial, values);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const float up_x = ldexpf(1.f, sc.ex), up_a = ldexpf(1.f, sc.ea), up_b = ldexpf(1.f, sc.eb);
    normalize_kernel<<<dim3((l.nb + 3) / 4, (l.mb + 3) / 4, batch), 256, 0, stream>>>(g, type, partial, chunks, eps, up_x, x, xt[0], l.m, l.n,
                                                                                     l.mb, l.nb, tall, l.x_halves);
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
        if ((e = pair_gemm<GRAM>(k, batch, stream)) != hipSuccess) return e;
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
        if ((e = pair_gemm<POLYNOMIAL>(k, batch, stream)) != hipSuccess) return e;
        const bool last = s == steps - 1;
        k.p = b;
        k.q = xt[s & 1];
        k.out = last ? nullptr : x;
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
        if ((e = pair_gemm<APPLY>(k, batch, stream)) != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace cake
