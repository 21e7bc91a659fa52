// out = residual + act(x w^T + bias) with x and w in float32 (epilogue.cuh says what follows the product): products and sums are float32
// multiply-adds, no reduced-precision matrix mode.
//
// A warp holds the whole tile of its CTA, 4 TN rows of x by 8 TM rows of w, for a share of K: the blocks of 16 of K go round the warps of
// the CTA and, where there are few tiles, of a cluster of CTAs, each warp with a ring of its own that it fills by cp.async and nobody else
// waits for.  The warps' parts are added at the end, in their order, through shared memory and the cluster's.  So a thread has up to 8 x 8
// sums although a CTA's tile is small enough for every SM to have some, and reads 16 bytes of shared memory per 16 multiply-adds.  What part
// of K a warp has depends on K and on the rows of w: a row of x has the same bits whatever rows are beside it.
// What bounds it: many rows, the main loop, which takes 55 % of the multiply-adds that the pipe's width says (a 24 x 64 tile 11.3 us per 1,024 of
// K; the plain product's 64 x 128 tile, which reads shared memory half as often for a multiply-add, has 78 %), and the tiles' ends, 1.6 us each in
// which an SM's half multiplies nothing: 301 x 2,048 x 1,024 49 us, of which 17.5 at the full width and some 9 the ends of its six tiles an SM (832
// CTAs over 296 places; the multiply-add pipe is busy for 44 % of the time); the plain product's form with tiles that every warp shares 54.  Few
// rows, the weights (1 x 12,288 x 4,096 45 us, 4.4 TB/s); few of everything, the latency of a ring's first turn and the join (1 x 155 x 9,596
// 14 us, one chain over K 49).
// Each sum is a pair, of the even k and of the odd ones, so that packed multiply-adds take the operands as they lie in memory; a chain then is
// K over twice the warps long, and rounds less than one over all of K.
// Lanes are dealt so that neighbours share a row of one operand or of the other (bits 0 and 4 pick the row of x, bits 1 to 3 that of w).
#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "epilogue.cuh"
#include "packed.cuh"
#include "tc_product.cuh"

namespace iian {

constexpr int LN_DEPTH = 16, LN_LD = LN_DEPTH + 4;           // rows 20 floats apart: 16-byte reads of 8 neighbouring rows hit 32 banks

// PIECE floats to shared memory, zeros where there are none; PIECE 1: rows that do not begin on 16 bytes
template <int PIECE> __device__ __forceinline__ void ln_copy(float * to, const float * from, bool there) {
    if constexpr (PIECE == 4) copy16(to, from, there);
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"((unsigned) __cvta_generic_to_shared(to)), "l"(from), "r"(there ? 4 : 0));
}

template <int TN, int TM, int WARPS, int STAGES, int PIECE>
__global__ void __launch_bounds__(WARPS * 32)
linear_f32_kernel(const float * __restrict__ x, long long ldx, const float * __restrict__ w, int N, int M, int K, int row_tiles, int ks, const LinearEpilogue epi) {
    constexpr int ROWS = 4 * TN, COLS = 8 * TM, ALL = ROWS + COLS, PLD = COLS + 8, PIECES = LN_DEPTH / PIECE, STEP = 32 / PIECES;
    static_assert(ROWS % STEP == 0 && COLS % STEP == 0, "a step of the loader lies in x or in w as a whole");
    static_assert(WARPS * ROWS * PLD <= WARPS * STAGES * ALL * LN_LD, "the parts take the rings' place");
    extern __shared__ __align__(16) float smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int rank = blockIdx.x % ks, tile = blockIdx.x / ks;                    // a cluster is ks neighbours
    const int n0 = tile % row_tiles * ROWS, m0 = tile / row_tiles * COLS;
    const int blocks = (K + LN_DEPTH - 1) / LN_DEPTH, unit = rank * WARPS + warp, units = ks * WARPS;
    const int turns = blocks > unit ? (blocks - unit + units - 1) / units : 0;
    float * ring = smem + warp * (STAGES * ALL * LN_LD);
    // where the lane's pieces come from: STEP rows apart; zeros behind the last row of x, and behind w's the last one again (nobody reads what
    // comes of that)
    const int at = lane % PIECES * PIECE, first = lane / PIECES;
    const float * xb = x + (long long) min(n0 + first, N - 1) * ldx + at, * wb = w + (long long) min(m0 + first, M - 1) * K + at;
    const unsigned x_step = (unsigned) ldx * STEP, w_step = (unsigned) K * STEP;
    const int x_rows = N - n0 - first;
    const unsigned w_last = max(M - 1 - m0 - first, 0) / STEP;
    auto fill = [&](int s) {
        if (s < turns) {
            const int k = (unit + s * units) * LN_DEPTH;
            const bool in = k + at < K;                      // K is a multiple of PIECE: a piece lies inside or outside as a whole
            const float * xs = xb + (in ? k : -at), * ws = wb + (in ? k : -at);
            float * to = ring + (s % STAGES * ALL + first) * LN_LD + at;
#pragma unroll
            for (int i = 0; i < ROWS / STEP; i++) ln_copy<PIECE>(to + i * STEP * LN_LD, in && i * STEP < x_rows ? xs + (unsigned long long) i * x_step : x, in && i * STEP < x_rows);
#pragma unroll
            for (int i = 0; i < COLS / STEP; i++)
                ln_copy<PIECE>(to + (ROWS + i * STEP) * LN_LD, ws + (unsigned long long) min((unsigned) i, w_last) * w_step, in);
        }
        asm volatile("cp.async.commit_group;");
    };
#pragma unroll
    for (int s = 0; s < STAGES - 1; s++) fill(s);
    unsigned long long acc[TN][TM];
#pragma unroll
    for (int i = 0; i < TN; i++)
#pragma unroll
        for (int j = 0; j < TM; j++) acc[i][j] = 0ull;
    const int row = (lane & 1) | (lane >> 4) << 1, col = (lane >> 1) & 7;
    for (int s = 0; s < turns; s++) {
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
        __syncwarp();                                        // this stage has landed for every lane; the one before has been read by every lane
        fill(s + STAGES - 1);
        const float * xr = ring + (s % STAGES * ALL + row) * LN_LD, * wr = ring + (s % STAGES * ALL + ROWS + col) * LN_LD;
#pragma unroll
        for (int k = 0; k < LN_DEPTH; k += 4) {
            ulonglong2 a[TN], b[TM];
#pragma unroll
            for (int i = 0; i < TN; i++) a[i] = *reinterpret_cast<const ulonglong2 *>(xr + i * 4 * LN_LD + k);
#pragma unroll
            for (int j = 0; j < TM; j++) b[j] = *reinterpret_cast<const ulonglong2 *>(wr + j * 8 * LN_LD + k);
#pragma unroll
            for (int i = 0; i < TN; i++)
#pragma unroll
                for (int j = 0; j < TM; j++) acc[i][j] = fma2(a[i].x, b[j].x, acc[i][j]);
#pragma unroll
            for (int i = 0; i < TN; i++)
#pragma unroll
                for (int j = 0; j < TM; j++) acc[i][j] = fma2(a[i].y, b[j].y, acc[i][j]);
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();                                         // every warp is done with its ring: the parts take the place
#pragma unroll
    for (int i = 0; i < TN; i++)
#pragma unroll
        for (int j = 0; j < TM; j++) {
            const float2 v = unpack2(acc[i][j]);
            smem[(warp * ROWS + row + 4 * i) * PLD + col + 8 * j] = v.x + v.y;
        }
    __syncthreads();
    auto put = [&](int r, int c, float4 v) {                 // 4 columns from c on of row r
        const int live = M - m0 - c;
        if (n0 + r >= N || live <= 0) return;
        const float4 b = epi.bias4(m0 + c, live), d = epi.residual4((size_t) (n0 + r), m0 + c, live);
        float y[4] = {v.x + b.x, v.y + b.y, v.z + b.z, v.w + b.w};
        linear_act_values<4>(y, epi.act);
        if (epi.res != nullptr) { y[0] += d.x; y[1] += d.y; y[2] += d.z; y[3] += d.w; }
        epi.put4(y, (size_t) (n0 + r), m0 + c, live);
    };
    constexpr int GROUPS = WARPS / 4;                        // four warps' parts first, then those of all groups in their order, whoever holds them
    auto add = [](float4 & v, const float4 & u) { v.x += u.x; v.y += u.y; v.z += u.z; v.w += u.w; };
    for (int e = threadIdx.x; e < ROWS * COLS / 4; e += WARPS * 32) {
        const int r = e / (COLS / 4), c = e % (COLS / 4) * 4;
        float4 v[GROUPS];
#pragma unroll
        for (int g = 0; g < GROUPS; g++) {
            v[g] = *reinterpret_cast<const float4 *>(smem + (g * 4 * ROWS + r) * PLD + c);
#pragma unroll
            for (int p = 1; p < 4; p++) add(v[g], *reinterpret_cast<const float4 *>(smem + ((g * 4 + p) * ROWS + r) * PLD + c));
        }
        if (ks > 1) {
#pragma unroll
            for (int g = 0; g < GROUPS; g++) *reinterpret_cast<float4 *>(smem + (g * 4 * ROWS + r) * PLD + c) = v[g];
        } else {
#pragma unroll
            for (int g = 1; g < GROUPS; g++) add(v[0], v[g]);
            put(r, c, v[0]);
        }
    }
    if (ks > 1) {
        __syncthreads();
        cluster_sync_all();                                  // the parts of all of the cluster's CTAs lie there
        const unsigned base = (unsigned) __cvta_generic_to_shared(smem);
        for (int e = threadIdx.x + rank * WARPS * 32; e < ROWS * COLS / 4; e += ks * WARPS * 32) {
            const int r = e / (COLS / 4), c = e % (COLS / 4) * 4;
            float4 v;
            for (int p = 0; p < ks; p++) {
#pragma unroll
                for (int g = 0; g < GROUPS; g++) {
                    float4 u;
                    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(u.x), "=f"(u.y), "=f"(u.z), "=f"(u.w)
                                 : "r"(map_to_cta(base + ((g * 4 * ROWS + r) * PLD + c) * 4, p)) : "memory");
                    if (p == 0 && g == 0) v = u;
                    else add(v, u);
                }
            }
            put(r, c, v);
        }
        __syncwarp();
        cluster_sync_all();                                  // nobody leaves while its part is read
    }
}

template <int TN, int TM, int WARPS, int STAGES, int PIECE>
static int ln_launch(const float * x, long long ldx, const float * w, int N, int M, int K, int ks, const LinearEpilogue & epi, cudaStream_t stream) {
    constexpr size_t smem = (size_t) WARPS * STAGES * (4 * TN + 8 * TM) * LN_LD * sizeof(float);
    static_assert(smem <= 227 * 1024, "the rings fit");
    auto kernel = linear_f32_kernel<TN, TM, WARPS, STAGES, PIECE>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int) smem);
    if (e != cudaSuccess) return 1000 + (int) e;
    const long long row_tiles = (N + 4 * TN - 1) / (4 * TN), tiles = row_tiles * ((M + 8 * TM - 1) / (8 * TM));
    if (tiles * ks > 2147483647LL) return IIAN_ERR_LIMIT;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ks; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned) (tiles * ks)); cfg.blockDim = dim3(WARPS * 32); cfg.dynamicSmemBytes = smem; cfg.stream = stream;
    cfg.attrs = attr; cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, kernel, x, ldx, w, N, M, K, (int) row_tiles, ks, epi);
    return e == cudaSuccess ? iian_launch_status() : 1000 + (int) e;
}

// Over how many groups of four warps K goes: by K and the rows of w alone, so that a row's sums are those of any other number of rows.  Few
// rows of w leave SMs idle that could share K (1 x 155 x 9,596 14 us in eight groups, 38 in two), long K makes up for the join, short K does not
// even for a second group's (1,300 x 1,500 x 700 86 us in one, 99 in two), unless there are few rows of w besides.
static int ln_groups(int M, int K) {
    if (K < 768) return M < 1024 ? 2 : 1;
    return 2 * std::min(M < 1024 ? 4 : M < 4096 ? 2 : 1, K >= 4 * 768 ? 4 : K >= 2 * 768 ? 2 : 1);
}

// The tiles: rows of x, rows of w, warps, and us as measured (1 to 2,048 rows, K 256 to 11,264): of a launch, per 1,024 of K for the first
// tile of an SM and for each further one, of a tile's end, and of a cluster's join.
struct LnTile { int rows, cols, warps; double launch, first, further, end, join; };
constexpr LnTile LN_TILES[] = {{32, 64, 4, 2.2, 18.2, 14.3, 1.6, 2.0}, {24, 64, 4, 1.9, 15.1, 11.3, 1.6, 2.2}, {16, 64, 4, 1.6, 13.0, 8.8, 1.6, 2.2},
                               {16, 32, 8, 2.1, 6.1, 4.6, 1.5, 1.5}, {8, 32, 8, 1.8, 4.3, 3.2, 1.4, 2.2}};

static int ln_plan(int N, int M, int K, int groups, int sms) {
    int tile = 0;
    double best = 1e300;
    for (int v = 0; v < 5; v++) {
        const LnTile & p = LN_TILES[v];
        if (groups * 4 % p.warps != 0) continue;
        const int ks = groups * 4 / p.warps;
        const double tiles = (double) ((N + p.rows - 1) / p.rows) * ((M + p.cols - 1) / p.cols);
        const double slots = ks > 4 ? sms - sms / 9 : sms;               // clusters of eight leave some SMs of a GPC over
        const double turns = std::ceil(tiles * ks / slots);
        const double t = p.launch + turns * p.end + K / 1024.0 / ks * (p.first + p.further * (turns - 1)) + (ks > 1 ? p.join : 0.0);
        if (t < best) { best = t; tile = v; }
    }
    return tile;
}

template <int PIECE>
static int ln_go(int tile, const float * x, long long ldx, const float * w, int N, int M, int K, int ks, const LinearEpilogue & epi, cudaStream_t stream) {
    switch (tile) {
        case 0: return ln_launch<8, 8, 4, 3, PIECE>(x, ldx, w, N, M, K, ks, epi, stream);
        case 1: return ln_launch<6, 8, 4, 3, PIECE>(x, ldx, w, N, M, K, ks, epi, stream);
        case 2: return ln_launch<4, 8, 4, 4, PIECE>(x, ldx, w, N, M, K, ks, epi, stream);
        case 3: return ln_launch<4, 4, 8, 3, PIECE>(x, ldx, w, N, M, K, ks, epi, stream);
        case 4: return ln_launch<2, 4, 8, 4, PIECE>(x, ldx, w, N, M, K, ks, epi, stream);
    }
    return IIAN_ERR_SHAPE;
}

}  // namespace iian

using namespace iian;

// The form of a product with M of a matrix's `of` rows that gives the bits which the product with all of them does.
IIAN_API int iian_linear_act_f32_form(int N, int M, int of, int K) {
    if (N <= 0 || M <= 0 || of < M || K <= 0) return 0;
    const int groups = ln_groups(of, K);
    return ln_plan(N, M, K, groups, 148) + 1 | groups << 8;
}

// x rows ldx apart; form 0: the tile and the groups of warps that suit the sizes, else tile + 1 | groups << 8
IIAN_API int iian_linear_act_f32(const float * x, long long ldx, const float * w, const float * bias, const void * residual, int res_dtype,
                                 long long ldr, void * out, int out_dtype, long long ldo, int N, int M, int K, int act, int form, cudaStream_t stream) {
    if (N <= 0 || M <= 0) return IIAN_OK;
    if (K <= 0 || ldx < K) return IIAN_ERR_SHAPE;
    // places behind the last one, and eight rows on, are 32-bit numbers too
    if (std::max(N, M) > 2147483647 - 1024 || std::max<long long>(K, ldx) >= 1LL << 29) return IIAN_ERR_LIMIT;
    LinearEpilogue e;
    if (!linear_epilogue(e, bias, residual, res_dtype, ldr, out, out_dtype, ldo, act)) return IIAN_ERR_DTYPE;
    const bool whole = K % 4 == 0 && ldx % 4 == 0 && ((uintptr_t) x | (uintptr_t) w) % 16 == 0;
    const int groups = form == 0 ? ln_groups(M, K) : form >> 8, tile = form == 0 ? ln_plan(N, M, K, groups, 148) : (form & 255) - 1;
    if (tile < 0 || tile > 4 || groups < 1 || groups > 8 || groups * 4 % LN_TILES[tile].warps != 0) return IIAN_ERR_SHAPE;
    const int ks = groups * 4 / LN_TILES[tile].warps;
    return whole ? ln_go<4>(tile, x, ldx, w, N, M, K, ks, e, stream) : ln_go<1>(tile, x, ldx, w, N, M, K, ks, e, stream);
}
