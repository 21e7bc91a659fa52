// Matrix products of bfloat16 rows with what follows them in their epilogue, on tcgen05 (tc_product.cuh):
//
//   iian_linear_act       out[t, n] = residual[t, n] + act(sum_k x[t, k] w[n, k] + bias[n])
//   iian_linear_logprobs  z[t, v] = sum_k x[t, k] w[v, k] (capped: c tanh(z / c));  lse[t] = log sum_v exp z[t, v];
//                         lp[t] = z[t, target[t]] - lse[t]          -- the logits are never written
//
// A tile is 128 rows of x on one SM, or 256 on a pair of SMs, times bn rows of w (bn is chosen per call: a multiple of 16, on pairs of 32,
// up to 256).  Warp 0 brings both operands by TMA, K in blocks of 64, warp 1 multiplies, warps 2..5 run the epilogue on a thread's own
// row of the accumulator while the next tile is multiplied into the other one.
//
// Few rows of x: the rows of w are the product's and those of x its columns (SWAP), up to 128 of w a tile and all of x, in sixteens.  The
// accumulator then has a row of w in a lane: the epilogue turns it around in shared memory, the softmax's sums are taken over the lanes.
// Where x's rows stay the product's although there are fewer than 128, a stage holds only those there are (in eights).  In either case a tile
// may have fewer rows than the 128 that the product reads of shared memory; what lies behind the real ones only reaches rows of the
// accumulator that nobody reads.
//
// Few tiles: the K blocks of a tile are shared by a cluster of `ks` CTAs.  Each sends its part into the others' shared memory, and each adds up
// all parts, in their order, for its share of the tile.  Nothing is sent before every CTA of the cluster has begun: on pairs the barrier at the
// start says so, single CTAs arrive at one there and wait for it before they send, when the products are long done.
//
// The softmax's sums: a thread walks its row's columns with a running maximum and sum and leaves them per tile; a second kernel joins a
// row's.  The maximum is the running one, so no exponential overflows; an empty sum has the maximum minus infinity.
//
// Launches are programmatic (common.cuh): set-up runs beside the end of the kernel before (1 x 4,096 x 1,024 8.2 -> 5.7 us).  None announces its
// own successor early: the joins of scores that were then let in while the product ran cost it 40 to 60 us of 200 (16 and 61 rows), and
// products gain nothing by it.
//
// Every wait is bounded, as in gemm_tcgen05.cu; a producer that gives up waits, bounded too, for the copies it still has under way.
#include <math_constants.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "epilogue.cuh"
#include "tc_product.cuh"

namespace iian {

constexpr int LF_STAGES = 24;             // barriers there are; how many are used follows from the size of a stage
constexpr int LF_WARPS = 8;               // epilogue warps: two for each quarter of the accumulator's lanes, sharing its columns
constexpr int LF_THREADS = 64 + 32 * LF_WARPS;
constexpr int LF_COLS = 16;               // columns an epilogue warp turns around at a time; rows of 64 bytes, their 16-byte pieces swapped so that
                                          // neither writing a row a lane nor reading two rows by eight lanes meets a bank twice
constexpr int LF_TURN = 128 / LF_COLS, LF_TURNS = 32 / LF_TURN;       // rows a warp's access covers, and accesses for 32 rows
constexpr int kLfRing = 208 * 1024, kLfSmem = kLfRing + LF_WARPS * 32 * LF_COLS * 4 + 1024;
constexpr float kLog2e = 1.4426950408889634f;

struct LfScore {
    float2 * part;                        // [2 column tiles][T]: maximum and sum of a row's columns in a tile, of one warp's and of the other's
    const int * targets;
    float * lp;                           // receives the target's logit
    float cap;                            // 0: none
};

// What follows the product.  LF_ANY takes every type, place and width an entry at a time where it has to; the four others have their types fixed
// and every access of 4 columns whole and aligned, so that nothing is decided between the sums and the store (2,048 x 4,096 outputs behind a
// K of 64, which is all epilogue: 18 us with the decisions).
enum { LF_SCORE = 0, LF_ANY = 1, LF_BF16 = 2, LF_F32 = 3, LF_BF16_RES = 4, LF_F32_RES = 5 };       // (the residual of the last two is float32)

struct LfArgs {
    int T, N, bn, ks, x_cols, stages, stage_bytes, a_bytes, kb_bytes, all_kb, m_tiles, num_tiles, units;
    // where K is shared: a CTA adds up `per` of the tile's groups of 4 columns (inv_per = 65536 / per, rounded up); the parts arrive at
    // recv_off, rows of recv_ld groups for every CTA that sends, over the ring (recv_shared) or behind it
    int per, inv_per, recv_off, recv_ld, recv_rows, recv_shared;
    // a tile's K blocks go to `accs` accumulators in turn, added up in the epilogue: the sums in tensor memory are not rounded but cut off, so
    // that the error grows with the length of the chain, and products into one accumulator wait for one another (90 ns each however few
    // columns they have); buf_cols: columns of all of them.  Tiles of 256 columns leave room for one (2,048 x 12,288 x 4,096 in bfloat16 differs
    // from sums in float32 by 1.6e-4 of its norm, a tenth of what the rounding of the outputs does, and 2,048 scores by 6e-7)
    int accs, buf_cols;
    unsigned tmem_cols;
    TcStatus * status;
    LinearEpilogue epi;
    LfScore score;
};

__device__ __forceinline__ float lf_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float lf_finite_or_zero(float m) { return fabsf(m) < CUDART_INF_F ? m : 0.0f; }
// c tanh(z / c) within 2.2 units of 2^-22 of its value, for the sums and for the target's logit.  From |u| = 0.8 on, u = z / c, it is c (1 - 2 / (1 +
// e^2u)) with the hardware's exponential, whose difference would lose the digits of small u (1e-4 at a cap of 1,000); below, z times a polynomial
// in u^2 (minimax for tanh(u) / u, 4e-9).
__device__ __forceinline__ float lf_capped(float z, float cap, float inv_cap) {
    const float u = z * inv_cap, v = u * u, zv = z * v;
    const float q = __fdividef(2.0f, 1.0f + lf_exp2(2.8853900817779268f * fabsf(u)));
    float t = fmaf(v, 0.0015676724f, -0.007374115f);
    t = fmaf(v, t, 0.02127475f);
    t = fmaf(v, t, -0.053841557f);
    t = fmaf(v, t, 0.13332023f);
    t = fmaf(v, t, -0.3333328f);
    return fabsf(u) < 0.8f ? fmaf(zv, t, z) : copysignf(cap * (1.0f - q), z);
}

// LF_COLS columns of 32 lanes
__device__ __forceinline__ void lf_ld(unsigned taddr, unsigned * r) {
    static_assert(LF_COLS == 16, "");
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                   "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr) : "memory");
}

// the same of a tile's accumulators together, `between` columns apart
__device__ __forceinline__ void lf_sum(unsigned taddr, int accs, int between, float * y) {
    unsigned r[LF_COLS];
    lf_ld(taddr, r);
    tc_wait_ld();
#pragma unroll
    for (int i = 0; i < LF_COLS; i++) y[i] = __uint_as_float(r[i]);
    for (int a = 1; a < accs; a++) {
        lf_ld(taddr + (unsigned) (a * between), r);
        tc_wait_ld();
#pragma unroll
        for (int i = 0; i < LF_COLS; i++) y[i] += __uint_as_float(r[i]);
    }
}

// LF_COLS columns of 32 lanes turned around: `turn` holds a column's 32 lanes side by side afterwards.  A whole warp calls it.
__device__ __forceinline__ void lf_turn(unsigned taddr, int accs, int between, float * turn, int lane) {
    float r[LF_COLS];
    lf_sum(taddr, accs, between, r);
    __syncwarp();                                            // the columns before have been read
#pragma unroll
    for (int j = 0; j < LF_COLS; j++) turn[j * 32 + lane] = r[j];
    __syncwarp();
}

// One value of 32 columns in every lane becomes, in lane c, column c's value over all lanes.
template <typename OP> __device__ __forceinline__ float lf_over_lanes(float (&v)[32], int lane, OP op) {
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1)
#pragma unroll
        for (int i = 0; i < o; i++) {
            const bool up = lane & o;
            const float send = up ? v[i] : v[i + o], keep = up ? v[i + o] : v[i];
            v[i] = op(keep, __shfl_xor_sync(0xffffffffu, send, o));
        }
    return v[0];
}

// 32 columns of a row, `live` of them in the matrix, into the row's running maximum and sum
__device__ __forceinline__ void lf_take(const unsigned * r, int live, float cap, float inv_cap, float & m, float & s) {
    float z[32], mx[4] = {-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
    for (int i = 0; i < 32; i++) {
        z[i] = __uint_as_float(r[i]);
        if (cap != 0.0f) z[i] = lf_capped(z[i], cap, inv_cap);
        if (i >= live) z[i] = -CUDART_INF_F;
        mx[i & 3] = fmaxf(mx[i & 3], z[i]);
    }
    const float m1 = fmaxf(fmaxf(m, fmaxf(mx[0], mx[1])), fmaxf(mx[2], mx[3])), ref = lf_finite_or_zero(m1) * kLog2e;
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 32; i++) sum[i & 3] += lf_exp2(fmaf(z[i], kLog2e, -ref));
    s = (s == 0.0f ? 0.0f : s * lf_exp2(fmaf(m, kLog2e, -ref))) + ((sum[0] + sum[1]) + (sum[2] + sum[3]));
    m = m1;
}

// r[at] without an address: registers have none, and an indexed copy in local memory would be written for every 32 columns
__device__ __forceinline__ unsigned lf_pick(const unsigned * r, int at) {
    unsigned v = 0;
#pragma unroll
    for (int i = 0; i < 32; i++) asm("{\n .reg .pred p;\n setp.eq.s32 p, %1, %2;\n @p mov.b32 %0, %3;\n}" : "+r"(v) : "r"(at), "r"(i), "r"(r[i]));
    return v;
}

template <int KIND> __device__ __forceinline__ float4 lf_residual(const LinearEpilogue & e, size_t row, int col, int live) {
    if constexpr (KIND == LF_ANY) return e.residual4(row, col, live);
    else if constexpr (KIND == LF_BF16_RES || KIND == LF_F32_RES)
        return live > 0 ? *reinterpret_cast<const float4 *>((const float *) e.res + row * (size_t) e.ldr + col) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    else return make_float4(0.0f, 0.0f, 0.0f, 0.0f);
}
template <int KIND> __device__ __forceinline__ float4 lf_bias(const LinearEpilogue & e, int col, int live) {
    if constexpr (KIND == LF_ANY) return e.bias4(col, live);
    else return e.bias != nullptr && live > 0 ? __ldg(reinterpret_cast<const float4 *>(e.bias + col)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
}
template <int KIND> __device__ __forceinline__ void lf_put(const LinearEpilogue & e, const float * y, const float4 & r, size_t row, int col, int live) {
    float v[4] = {y[0] + r.x, y[1] + r.y, y[2] + r.z, y[3] + r.w};
    if constexpr (KIND == LF_ANY) e.put4(v, row, col, live);
    else if (live > 0) {
        const size_t at = row * (size_t) e.ldo + col;
        if constexpr (KIND == LF_BF16 || KIND == LF_BF16_RES) {
            __nv_bfloat162 h[2] = {__floats2bfloat162_rn(v[0], v[1]), __floats2bfloat162_rn(v[2], v[3])};
            *reinterpret_cast<uint2 *>((__nv_bfloat16 *) e.out + at) = *reinterpret_cast<uint2 *>(h);
        } else *reinterpret_cast<float4 *>((float *) e.out + at) = make_float4(v[0], v[1], v[2], v[3]);
    }
}

// KPS: blocks of K a stage (two on pairs of SMs, one or two otherwise)
template <bool PAIR, bool SWAP, int KPS, int KIND>
__global__ void __launch_bounds__(LF_THREADS, 1) linear_fused_kernel(const __grid_constant__ CUtensorMap map_a,
                                                                     const __grid_constant__ CUtensorMap map_b, const LfArgs p) {
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char * smem = (unsigned char *) (((uintptr_t) smem_raw + 1023) & ~(uintptr_t) 1023);
    constexpr bool SCORE = KIND == LF_SCORE;
    constexpr int ROWS = PAIR ? 2 * TC_BM : TC_BM;
    __shared__ __align__(8) unsigned long long full_bar[LF_STAGES], empty_bar[LF_STAGES], acc_full[2], acc_empty[2];
    __shared__ unsigned tmem_base_s;

    const int warp = __shfl_sync(0xffffffffu, (int) threadIdx.x >> 5, 0), lane = threadIdx.x & 31;        // (uniform, and known to be)
    const int bn = p.bn, half = PAIR ? bn / 2 : bn, stages = p.stages, m_tiles = p.m_tiles, num_tiles = p.num_tiles, units = p.units;
    const unsigned cluster_rank = PAIR || p.ks > 1 ? cluster_cta_rank() : 0u;
    const unsigned rank = PAIR ? cluster_rank & 1u : 0u, leader = PAIR ? cluster_rank & ~1u : 0u;       // which CTA of a pair, and its first
    const int split = (int) (PAIR ? cluster_rank >> 1 : cluster_rank);        // which share of K
    const int block = PAIR ? (int) blockIdx.x >> 1 : (int) blockIdx.x, unit = p.ks > 1 ? block / p.ks : block;
    const int a_bytes = p.a_bytes, kb_bytes = p.kb_bytes;
    const int kb0 = p.ks > 1 ? p.all_kb * split / p.ks : 0, kb1 = p.ks > 1 ? p.all_kb * (split + 1) / p.ks : p.all_kb;
    const int acc_cols = ((SWAP ? p.x_cols : bn) + 31) & ~31;
    const int early = PAIR || unit >= num_tiles ? 0 : min(stages, kb1 - kb0);  // copies that are asked for before anything else is set up

    auto copy = [&](int s, int kb, int ya, int yb) {
        const unsigned to = smem_addr(smem + s * p.stage_bytes);
        if constexpr (PAIR) {
            const unsigned bar = map_to_cta(smem_addr(&full_bar[s]), leader);
            if (rank == 0) mbar_expect_tx_warp(smem_addr(&full_bar[s]), 2 * KPS * kb_bytes);
#pragma unroll
            for (int j = 0; j < KPS; j++) {
                tma_load_2d_pair_warp(to + j * kb_bytes, &map_a, (kb * KPS + j) * TC_BK, ya, bar);
                tma_load_2d_pair_warp(to + j * kb_bytes + a_bytes, &map_b, (kb * KPS + j) * TC_BK, yb, bar);
            }
        } else {
            const unsigned bar = smem_addr(&full_bar[s]);
            mbar_expect_tx_warp(bar, KPS * (SWAP ? (p.bn + p.x_cols) * TC_BK * 2 : kb_bytes));
#pragma unroll
            for (int j = 0; j < KPS; j++) {
                tma_load_2d_warp(to + j * kb_bytes, &map_a, (kb * KPS + j) * TC_BK, ya, bar);
                tma_load_2d_warp(to + j * kb_bytes + a_bytes, &map_b, (kb * KPS + j) * TC_BK, yb, bar);
            }
        }
    };

    if (warp == 0) {
        if (lane == 0) {
            for (int s = 0; s < stages; s++) { mbar_init(smem_addr(&full_bar[s]), 1); mbar_init(smem_addr(&empty_bar[s]), 1); }
            for (int b = 0; b < 2; b++) { mbar_init(smem_addr(&acc_full[b]), 1); mbar_init(smem_addr(&acc_empty[b]), PAIR ? 2 * LF_WARPS : LF_WARPS); }
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        __syncwarp();
        pdl_wait();
        for (int i = 0; i < early; i++) copy(i, kb0 + i, SWAP ? unit * bn : unit % m_tiles * ROWS, SWAP ? 0 : unit / m_tiles * bn);
    }
    if (warp == 1) {
        if constexpr (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_base_s)), "r"(p.tmem_cols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_base_s)), "r"(p.tmem_cols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    tc_fence_before();
    __syncthreads();
    pdl_wait();                                   // set-up runs beside the end of the kernel before; nothing in memory is read or written until here
    if constexpr (PAIR) cluster_sync_all();       // the peer's barriers exist before anything arrives on them
    else if (p.ks > 1) {
        __syncwarp();
        cluster_arrive();                         // this CTA has begun: waited for before the parts are sent, on every way there
    }
    tc_fence_after();
    const unsigned tmem_base = tmem_base_s;

    if (warp == 0) {
        // ---- producer: stage s of the ring, in its `turn`-th use (no division: the loops below are chains of a few hundred cycles) --------
        int it = 0, s = 0;
        unsigned turn = 0;
        bool gave_up = false;
        for (int tile = unit; tile < num_tiles && !gave_up; tile += units) {
            const int ya = SWAP ? tile * bn : tile % m_tiles * ROWS + (int) rank * TC_BM, yb = SWAP ? 0 : tile / m_tiles * bn + (int) rank * half;
            for (int kb = kb0; kb < kb1; kb++, it++) {
                if (it >= early) {
                    if (!mbar_wait(smem_addr(&empty_bar[s]), (turn & 1) ^ 1)) { if (lane == 0) { p.status->code = 1; p.status->where = it; } gave_up = true; break; }
                    copy(s, kb, ya, yb);
                }
                if (++s == stages) { s = 0; turn++; }
            }
        }
        if (gave_up) {                            // its copies land before the CTA may leave
            if (rank == 0)
                for (int i = max(0, it - stages); i < it; i++) mbar_wait(smem_addr(&full_bar[i % stages]), (i / stages) & 1);
        } else if (PAIR) {                        // the last commits still arrive on this CTA's barriers
            for (int i = 0; i < stages; i++) {
                if (!mbar_wait(smem_addr(&empty_bar[s]), (turn & 1) ^ 1)) { if (lane == 0) { p.status->code = 5; p.status->where = it; } break; }
                if (++s == stages) { s = 0; turn++; }
            }
        }
    } else if (warp == 1 && rank == 0) {
        // ---- MMA issuer -------------------------------------------------------------------------------------
        const unsigned idesc = instr_desc_bf16(ROWS, SWAP ? p.x_cols : bn);
        const unsigned long long first = smem_desc_sw128(smem_addr(smem)), to_b = (unsigned long long) (a_bytes >> 4);
        const unsigned long long next_block = (unsigned long long) (kb_bytes >> 4), next_stage = (unsigned long long) (p.stage_bytes >> 4);
        unsigned long long at = first;            // (a ring of 208 KB: the descriptor's 14 bits of address do not overflow)
        int s = 0, use = 0;
        unsigned turn = 0;
        bool gave_up = false;
        for (int tile = unit; tile < num_tiles && !gave_up; tile += units, use++) {
            const int buf = use & 1;
            if (!mbar_wait(smem_addr(&acc_empty[buf]), ((use >> 1) & 1) ^ 1)) { if (lane == 0) { p.status->code = 4; p.status->where = use; } break; }
            tc_fence_after();
            const unsigned d_tmem = tmem_base + (unsigned) (buf * p.buf_cols);
            int a = 0;
            unsigned more = 0;                    // whether the accumulator already holds sums
            for (int kb = kb0; kb < kb1; kb++) {
                if (!mbar_wait(smem_addr(&full_bar[s]), turn & 1)) { if (lane == 0) { p.status->code = 2; p.status->where = kb; } gave_up = true; break; }
                tc_fence_after();
#pragma unroll
                for (int j = 0; j < KPS; j++) {
                    const unsigned long long da = at + j * next_block, db = da + to_b;
                    if constexpr (PAIR) tc_mma4_pair(d_tmem + (unsigned) (a * acc_cols), da, db, idesc, more);
                    else tc_mma4(d_tmem + (unsigned) (a * acc_cols), da, db, idesc, more);
                    if (++a == p.accs) { a = 0; more = 1; }
                }
                if constexpr (PAIR) tc_commit_pair_warp(smem_addr(&empty_bar[s]), leader);
                else tc_commit_warp(smem_addr(&empty_bar[s]));
                at += next_stage;
                if (++s == stages) { s = 0; turn++; at = first; }
            }
            if (!gave_up) {
                if constexpr (PAIR) tc_commit_pair_warp(smem_addr(&acc_full[buf]), leader);
                else tc_commit_warp(smem_addr(&acc_full[buf]));
            }
        }
    } else if (warp >= 2) {
        // ---- epilogue: warp w reads tensor-memory lanes 32 * (w % 4) .. + 31 -----------------------------------
        const int q = warp & 3, half_w = (warp - 2) >> 2;          // the second four warps take every other columns
        const float inv_cap = SCORE && p.score.cap != 0.0f ? 1.0f / p.score.cap : 0.0f;
        int use = 0;
        for (int tile = unit; tile < num_tiles; tile += units, use++) {
            const int buf = use & 1;
            const int n_tile = tile / m_tiles, m0 = tile % m_tiles * ROWS + (int) rank * TC_BM, n0 = n_tile * bn;
            const int row = m0 + q * 32 + lane, cols = min(bn, p.N - n0);
            if constexpr (!SCORE) {
                if (p.epi.res != nullptr && row < p.T) {          // the residual's lines come into the L2 while the products run
                    const int size = p.epi.res_bf16 ? 2 : 4;
                    const char * line = (const char *) p.epi.res + ((size_t) row * p.epi.ldr + n0) * size;
                    for (int b = half_w * 128; b < cols * size; b += 256) asm volatile("prefetch.global.L2 [%0];" ::"l"(line + b));
                }
            }
            if (!mbar_wait(smem_addr(&acc_full[buf]), (use >> 1) & 1)) {
                if (lane == 0) { p.status->code = 3; p.status->where = use; }
                break;
            }
            tc_fence_after();
            const unsigned acc = tmem_base + ((unsigned) (q * 32) << 16) + (unsigned) (buf * p.buf_cols);
            if constexpr (SWAP) {
                // a lane is a row of w, a column one of x
                const int limit = min(bn, p.N - n0) - q * 32;             // rows of w that this warp's lanes are
                if constexpr (SCORE) {
                    // a column's maximum and sum over the lanes: halves of the columns are handed from lane to lane until lane c has column c
#pragma unroll 1
                    for (int c0 = half_w * 32; c0 < p.T; c0 += 64) {
                        unsigned r[32];
                        tc_ld32(acc + (unsigned) c0, r);
                        tc_wait_ld();
                        if (p.accs == 2) {
                            unsigned r2[32];
                            tc_ld32(acc + (unsigned) (acc_cols + c0), r2);
                            tc_wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; i++) r[i] = __float_as_uint(__uint_as_float(r[i]) + __uint_as_float(r2[i]));
                        }
                        float z[32], v[32];
#pragma unroll
                        for (int i = 0; i < 32; i++) {
                            z[i] = __uint_as_float(r[i]);
                            if (p.score.cap != 0.0f) z[i] = lf_capped(z[i], p.score.cap, inv_cap);
                            if (lane >= limit) z[i] = -CUDART_INF_F;
                            v[i] = z[i];
                        }
                        const float m = lf_over_lanes(v, lane, [](float a, float b) { return fmaxf(a, b); });
                        const float ref = lf_finite_or_zero(m) * kLog2e;
#pragma unroll
                        for (int i = 0; i < 32; i++) v[i] = lf_exp2(fmaf(z[i], kLog2e, -__shfl_sync(0xffffffffu, ref, i)));
                        const float s = lf_over_lanes(v, lane, [](float a, float b) { return a + b; });
                        const int token = c0 + lane, wanted = token < p.T ? p.score.targets[token] : -1, rel = wanted < 0 ? -1 : wanted - n0 - q * 32;
                        if (token < p.T) p.score.part[((size_t) n_tile * 4 + q) * p.T + token] = make_float2(m, s);
                        unsigned here = __ballot_sync(0xffffffffu, rel >= 0 && rel < min(limit, 32));
                        while (here != 0) {                               // (a target among this warp's rows of w)
                            const int c = __ffs(here) - 1, from = __shfl_sync(0xffffffffu, rel, c);
                            const float x = __uint_as_float(lf_pick(r, c));
                            if (lane == from) p.score.lp[c0 + c] = p.score.cap != 0.0f ? lf_capped(x, p.score.cap, inv_cap) : x;
                            here &= here - 1;
                        }
                    }
                } else if (p.ks == 1 && limit > 0) {
                    float * turn = reinterpret_cast<float *>(smem + kLfRing) + (warp - 2) * 32 * LF_COLS;
                    const int in_row = lane / 8, in_col = lane % 8 * 4, col = n0 + q * 32 + in_col, live = limit - in_col;
                    const float4 bias = lf_bias<KIND>(p.epi, col, live);
#pragma unroll 1
                    for (int c0 = half_w * LF_COLS; c0 < p.T; c0 += 2 * LF_COLS) {
                        float4 res[4];
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const int token = c0 + in_row + 4 * i;
                            res[i] = lf_residual<KIND>(p.epi, (size_t) token, col, token < p.T ? live : 0);
                        }
                        lf_turn(acc + (unsigned) c0, p.accs, acc_cols, turn, lane);
                        float y[16];
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const float4 v = *reinterpret_cast<const float4 *>(turn + (in_row + 4 * i) * 32 + in_col);
                            y[4 * i] = v.x + bias.x; y[4 * i + 1] = v.y + bias.y; y[4 * i + 2] = v.z + bias.z; y[4 * i + 3] = v.w + bias.w;
                        }
                        linear_act_values<16>(y, p.epi.act);
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const int token = c0 + in_row + 4 * i;
                            lf_put<KIND>(p.epi, y + 4 * i, res[i], (size_t) token, col, token < p.T ? live : 0);
                        }
                    }
                }
            } else
            if (m0 + q * 32 < p.T) {              // (a warp whose rows are all behind the last one has nothing to do)
                if constexpr (SCORE) {
                    float m = -CUDART_INF_F, s = 0.0f;
                    const int wanted = row < p.T ? p.score.targets[row] : -1, target = wanted < 0 ? -1 : wanted - n0;
#pragma unroll 1
                    for (int c0 = half_w * 32; c0 < cols; c0 += 64) {
                        unsigned r[32];
                        tc_ld32(acc + (unsigned) c0, r);
                        tc_wait_ld();
                        if (p.accs == 2) {
                            unsigned r2[32];
                            tc_ld32(acc + (unsigned) (acc_cols + c0), r2);
                            tc_wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; i++) r[i] = __float_as_uint(__uint_as_float(r[i]) + __uint_as_float(r2[i]));
                        }
                        lf_take(r, cols - c0, p.score.cap, inv_cap, m, s);
                        if (target >= c0 && target < c0 + 32 && target < cols) {
                            const float z = __uint_as_float(lf_pick(r, target - c0));
                            p.score.lp[row] = p.score.cap != 0.0f ? lf_capped(z, p.score.cap, inv_cap) : z;
                        }
                    }
                    if (row < p.T) p.score.part[((size_t) n_tile * 2 + half_w) * p.T + row] = make_float2(m, s);
                } else if (p.ks == 1) {
                    // 32 rows of LF_COLS columns at a time, turned around in shared memory: a lane then holds 4 columns of every LF_TURN-th row, so
                    // that the residual is read and the result written whole lines at a time.  The residual is asked for before the sums.
                    float * turn = reinterpret_cast<float *>(smem + kLfRing) + (warp - 2) * 32 * LF_COLS;
                    const int in_row = lane / (LF_COLS / 4), in_col = lane % (LF_COLS / 4) * 4, row0 = m0 + q * 32;
                    auto residual = [&](int c0, float4 (&res)[LF_TURNS]) {
#pragma unroll
                        for (int i = 0; i < LF_TURNS; i++) {
                            const int r0 = row0 + in_row + i * LF_TURN;
                            res[i] = lf_residual<KIND>(p.epi, (size_t) r0, n0 + c0 + in_col, r0 < p.T ? cols - c0 - in_col : 0);
                        }
                    };
                    float4 res[LF_TURNS], next[LF_TURNS];
                    residual(half_w * LF_COLS, next);
#pragma unroll 1
                    for (int c0 = half_w * LF_COLS; c0 < cols; c0 += LF_WARPS / 4 * LF_COLS) {
                        const int live = cols - c0 - in_col, col = n0 + c0 + in_col;
#pragma unroll
                        for (int i = 0; i < LF_TURNS; i++) res[i] = next[i];
                        residual(c0 + LF_WARPS / 4 * LF_COLS, next);
                        const float4 bias = lf_bias<KIND>(p.epi, col, live);
                        float r[LF_COLS];
                        lf_sum(acc + (unsigned) c0, p.accs, acc_cols, r);
                        __syncwarp();                                   // the columns before have been read
#pragma unroll
                        for (int v = 0; v < LF_COLS / 4; v++)
                            *reinterpret_cast<float4 *>(turn + lane * LF_COLS + (v ^ ((lane >> 1) & 3)) * 4) = make_float4(r[4 * v], r[4 * v + 1], r[4 * v + 2], r[4 * v + 3]);
                        __syncwarp();
                        float y[4 * LF_TURNS];
#pragma unroll
                        for (int i = 0; i < LF_TURNS; i++) {
                            const float4 v = *reinterpret_cast<const float4 *>(turn + (in_row + i * LF_TURN) * LF_COLS + (in_col ^ (((in_row + i * LF_TURN) >> 1) & 3) * 4));
                            y[4 * i] = v.x + bias.x; y[4 * i + 1] = v.y + bias.y; y[4 * i + 2] = v.z + bias.z; y[4 * i + 3] = v.w + bias.w;
                        }
                        linear_act_values<4 * LF_TURNS>(y, p.epi.act);
#pragma unroll
                        for (int i = 0; i < LF_TURNS; i++) {
                            const int r0 = row0 + in_row + i * LF_TURN;
                            lf_put<KIND>(p.epi, y + 4 * i, res[i], (size_t) r0, col, r0 < p.T ? live : 0);
                        }
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if constexpr (PAIR) mbar_arrive_cluster(map_to_cta(smem_addr(&acc_empty[buf]), leader));
                else mbar_arrive(smem_addr(&acc_empty[buf]));
            }
        }
    }
    // ---- common exit: everybody arrives here, also after a wait that gave up -----------------------------------
    tc_fence_before();
    __syncthreads();
    __syncwarp();
    if constexpr (!SCORE) {
        if (p.ks > 1) {
            if constexpr (!PAIR) cluster_wait();              // every CTA of the cluster has begun: its shared memory may be written
            if (p.recv_shared) cluster_sync_all();            // every CTA's ring is done with
            const int m0 = unit % m_tiles * ROWS + (int) rank * TC_BM, n0 = unit / m_tiles * bn, rows = min(TC_BM, p.T - m0);
            const unsigned recv = smem_addr(smem) + (unsigned) p.recv_off;
            if (warp >= 2) {
                // this CTA's sums go to the CTAs that add them up, 4 columns a store; stores to another SM need no answer, where loads from there
                // waited a microsecond each time round (128 x 4,096 x 4,096 18.5 us)
                tc_fence_after();
                const int q = warp & 3, row = q * 32 + lane;
                const unsigned acc = tmem_base + ((unsigned) (q * 32) << 16), mine = recv + (unsigned) ((split * p.recv_rows + row) * p.recv_ld) * 16u;
                if constexpr (SWAP) {
                    float * turn = reinterpret_cast<float *>(smem + kLfRing) + (warp - 2) * 32 * LF_COLS;
                    const int in_row = lane / 8, i = q * 8 + lane % 8, owner = (i * p.inv_per) >> 16;
                    if (q * 32 < bn) {
#pragma unroll 1
                        for (int c0 = (warp - 2) / 4 * LF_COLS; c0 < rows; c0 += 2 * LF_COLS) {
                            lf_turn(acc + (unsigned) c0, p.accs, acc_cols, turn, lane);
#pragma unroll
                            for (int j = 0; j < 4; j++) {
                                const int token = c0 + in_row + 4 * j;
                                if (token < rows && 4 * i < bn) {
                                    const float4 v = *reinterpret_cast<const float4 *>(turn + (in_row + 4 * j) * 32 + lane % 8 * 4);
                                    const unsigned to = map_to_cta(recv + (unsigned) ((split * p.recv_rows + token) * p.recv_ld + i - owner * p.per) * 16u, (unsigned) owner);
                                    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
                                }
                            }
                        }
                    }
                } else if (q * 32 < rows) {
#pragma unroll 1
                    for (int c0 = (warp - 2) / 4 * LF_COLS; c0 < bn; c0 += LF_WARPS / 4 * LF_COLS) {
                        float r[LF_COLS];
                        lf_sum(acc + (unsigned) c0, p.accs, acc_cols, r);
                        if (row < rows) {
#pragma unroll
                            for (int v = 0; v < LF_COLS / 4; v++) {
                                const int i = c0 / 4 + v, owner = (i * p.inv_per) >> 16;
                                const unsigned to = map_to_cta(mine + (unsigned) (i - owner * p.per) * 16u, PAIR ? 2u * owner + rank : (unsigned) owner);
                                asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to), "f"(r[4 * v]), "f"(r[4 * v + 1]), "f"(r[4 * v + 2]), "f"(r[4 * v + 3]) : "memory");
                            }
                        }
                    }
                }
                tc_fence_before();
                __syncwarp();
            }
            cluster_sync_all();                               // all parts have arrived; nobody reaches into another's memory from here on
            const int from = split * p.per, width = min(p.per, (min(bn, p.N - n0) + 3) / 4 - from), pieces = width > 0 ? max(rows, 0) * width : 0;
            const float4 * part = reinterpret_cast<const float4 *>(smem + p.recv_off);
            for (int i = threadIdx.x; i < pieces; i += LF_THREADS) {
                const int row = i / width, c = i - row * width, col = n0 + (from + c) * 4, live = p.N - col;
                const float4 bias = lf_bias<KIND>(p.epi, col, live), res = lf_residual<KIND>(p.epi, (size_t) (m0 + row), col, live);
                float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                for (int r = 0; r < p.ks; r++) {
                    const float4 v = part[(r * p.recv_rows + row) * p.recv_ld + c];
                    y[0] += v.x; y[1] += v.y; y[2] += v.z; y[3] += v.w;
                }
                y[0] += bias.x; y[1] += bias.y; y[2] += bias.z; y[3] += bias.w;
                linear_act_values<4>(y, p.epi.act);
                lf_put<KIND>(p.epi, y, res, (size_t) (m0 + row), col, live);
            }
        }
    }
    if constexpr (PAIR) {
        if (p.ks == 1) cluster_sync_all();        // neither frees tensor memory or leaves while the other may use its memory
    }
    if (warp == 1) {
        tc_fence_after();
        if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(p.tmem_cols) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(p.tmem_cols) : "memory");
    }
}

// A row's maxima and sums of all column tiles become its log-sum-exp, the target's logit its log-probability.  A target below 0 is none: 0; one
// beyond the vocabulary is no number.  A CTA has JOIN_ROWS rows, a sector of each tile's line, and 128 threads for each: with 32 rows a CTA a few
// threads walked all of a row's tiles one behind the other (32 rows of 1,462 partial sums 30 us, now 4).
constexpr int JOIN_ROWS = 4;
__global__ void __launch_bounds__(512) logprobs_join_kernel(const float2 * __restrict__ part, int n_tiles, int T, int V,
                                                            const int * __restrict__ targets, float * __restrict__ lp, float * __restrict__ lse) {
    __shared__ float sm[512], ss[512];
    pdl_wait();
    constexpr int segs = 512 / JOIN_ROWS, rows = JOIN_ROWS;
    const int r = threadIdx.x % rows, seg = threadIdx.x / rows;
    const long long row = (long long) blockIdx.x * rows + r;
    float m = -CUDART_INF_F, s = 0.0f;
    auto add = [&](float m2, float s2) {
        const float m1 = fmaxf(m, m2), ref = lf_finite_or_zero(m1);
        s = (s == 0.0f ? 0.0f : s * lf_exp2((m - ref) * kLog2e)) + (s2 == 0.0f ? 0.0f : s2 * lf_exp2((m2 - ref) * kLog2e));
        m = m1;
    };
    if (row < T) {
#pragma unroll 8
        for (int i = seg; i < n_tiles; i += segs) m = fmaxf(m, part[(size_t) i * T + row].x);
        const float ref = lf_finite_or_zero(m);              // (differences first: where the maximum is one part's its factor is 1 exactly)
#pragma unroll 8
        for (int i = seg; i < n_tiles; i += segs) {
            const float2 v = part[(size_t) i * T + row];
            s += v.y == 0.0f ? 0.0f : v.y * lf_exp2((v.x - ref) * kLog2e);
        }
    }
    sm[threadIdx.x] = m;
    ss[threadIdx.x] = s;
    for (int o = segs / 2; o > 0; o >>= 1) {
        __syncthreads();
        if (seg < o) {
            add(sm[threadIdx.x + o * rows], ss[threadIdx.x + o * rows]);
            sm[threadIdx.x] = m;
            ss[threadIdx.x] = s;
        }
    }
    if (seg == 0 && row < T) {
        const float l = lf_finite_or_zero(m) + logf(s);
        const int t = targets[row];
        lse[row] = l;
        lp[row] = t < 0 ? 0.0f : t >= V ? CUDART_NAN_F : lp[row] - l;
    }
}

// Columns v0 .. v0 + P of the logits of T rows, as they lie in memory, into the rows' maxima and sums: a part for every `columns` of them, from
// part[first] on.  For element types and sizes that the tensor cores' product does not take.  Where a part begins and ends goes by the
// vocabulary alone, so that a row's sum has the same bits whatever rows are beside it.
__global__ void __launch_bounds__(256) logprobs_piece_kernel(const float * __restrict__ logits, int T, int P, int v0, const int * __restrict__ targets,
                                                             float * __restrict__ lp, float2 * __restrict__ part, int first, int columns, float cap) {
    __shared__ float sm[8], ss[8];
    pdl_wait();
    const size_t row = blockIdx.x;
    const int c0 = (int) blockIdx.y * columns, c1 = min(P, c0 + columns);
    const float * z = logits + row * P;
    float m = -CUDART_INF_F, s = 0.0f;
    auto add = [&](float m2, float s2) {
        const float m1 = fmaxf(m, m2), ref = lf_finite_or_zero(m1);
        s = (s == 0.0f ? 0.0f : s * expf(m - ref)) + (s2 == 0.0f ? 0.0f : s2 * expf(m2 - ref));
        m = m1;
    };
    for (int c = c0 + (int) threadIdx.x; c < c1; c += 256) {
        const float v = cap != 0.0f ? cap * tanhf(z[c] / cap) : z[c];
        if (v <= m) s += expf(v - lf_finite_or_zero(m));
        else add(v, 1.0f);                                   // (also what is no number: it becomes the sum)
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
        add(m2, s2);
    }
    const int warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) { sm[warp] = m; ss[warp] = s; }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < 8; i++) add(sm[i], ss[i]);
        part[(size_t) (first + blockIdx.y) * T + row] = make_float2(m, s);
        if (blockIdx.y == 0) {
            const int t = targets[row];
            if (t >= v0 && t - v0 < P) lp[row] = cap != 0.0f ? cap * tanhf(z[t - v0] / cap) : z[t - v0];
        }
    }
}

static int lf_join(const float * part, int n_tiles, int T, int V, const int * targets, float * lp, float * lse, cudaStream_t stream) {
    return iian_launch(logprobs_join_kernel, dim3((unsigned) ((T + JOIN_ROWS - 1) / JOIN_ROWS)), dim3(512), 0, stream, (const float2 *) part, n_tiles, T, V,
                       targets, lp, lse);
}

// SMs of the current device, asked for once
static int lf_sms() {
    static int known[64] = {};
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 148;
    if (dev >= 0 && dev < 64 && known[dev] > 0) return known[dev];
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) return 148;
    if (dev >= 0 && dev < 64) known[dev] = n;
    return n;
}

// T, N, bn, ks, status, epi or score as given; PAIR: tiles of 256 rows on pairs of SMs.
template <bool PAIR, bool SWAP, int KIND>
static int lf_launch(LfArgs & p, const void * x, long long ldx, const void * w, int K, int sms, cudaStream_t stream) {
    constexpr int ROWS = PAIR ? 2 * TC_BM : TC_BM;
    // All of it whatever the call needs: two CTAs of a cluster that each waited for the tensor memory of an SM's other CTA, those two in turn
    // waiting for their clusters, would never end, so no SM may hold two.
    constexpr int kRing = kLfRing, smem = kLfSmem, kRecvMost = 80 * 1024;
    if (SWAP && (p.T > TC_BM || p.bn > TC_BM)) return IIAN_ERR_SHAPE;
    p.x_cols = (p.T + 15) / 16 * 16;                                   // (SWAP: columns of the product; the rows behind the last are zeros)
    const int a_rows = SWAP ? (p.bn + 7) / 8 * 8 : PAIR || p.T >= TC_BM ? TC_BM : (p.T + 7) / 8 * 8, half = SWAP ? p.x_cols : PAIR ? p.bn / 2 : p.bn;
    p.a_bytes = a_rows * TC_BK * 2;
    p.kb_bytes = p.a_bytes + half * TC_BK * 2;
    const int over = (TC_BM - a_rows) * TC_BK * 2;                     // the last stage's product reads 128 rows too
    int ring = kRing;
    if (p.ks > 1) {
        p.per = (p.bn / 4 + p.ks - 1) / p.ks;
        p.inv_per = (65536 + p.per - 1) / p.per;
        p.recv_ld = p.per | 1;                                         // an odd number of 16-byte groups: rows of eight lanes meet no bank twice
        p.recv_rows = SWAP ? p.x_cols : a_rows;
        const int recv = p.ks * p.recv_rows * p.recv_ld * 16;
        if (recv > kRing) return IIAN_ERR_SHAPE;
        p.recv_shared = recv > kRecvMost;
        if (!p.recv_shared) ring = (kRing - recv) / 1024 * 1024;
        p.recv_off = p.recv_shared ? 0 : ring;
    }
    // two blocks of K a stage where four such stages fit and every share has two: a stage costs the warps that copy and multiply some 200 ns
    // whatever its size (128 x 128 x 16,384 55 us with one block a stage)
    const int blocks = (K + TC_BK - 1) / TC_BK, kps = PAIR || ((ring - over) / (2 * p.kb_bytes) >= 4 && blocks / 2 >= p.ks) ? 2 : 1;
    p.stage_bytes = kps * p.kb_bytes;
    p.stages = std::min(LF_STAGES, (ring - over) / p.stage_bytes);
    p.all_kb = (blocks + kps - 1) / kps;
    p.m_tiles = SWAP ? 1 : (p.T + ROWS - 1) / ROWS;
    const long long tiles = (long long) p.m_tiles * ((p.N + p.bn - 1) / p.bn);
    const int group = (PAIR ? 2 : 1) * p.ks;
    if (tiles * group > 2147483647LL - 65536) return IIAN_ERR_LIMIT;
    p.num_tiles = (int) tiles;
    p.units = p.ks > 1 ? p.num_tiles : std::min(p.num_tiles, sms / group);
    const int acc_cols = ((SWAP ? p.x_cols : p.bn) + 31) & ~31, bufs = p.units < p.num_tiles ? 2 : 1;      // (a CTA with one tile needs no second buffer)
    p.accs = 1;
    while (p.accs < (KIND == LF_SCORE ? 2 : 4) && 2 * p.accs * bufs * acc_cols <= 512 && 2 * p.accs <= p.all_kb / p.ks * kps) p.accs *= 2;
    p.buf_cols = p.accs * acc_cols;
    p.tmem_cols = 32;
    while (p.tmem_cols < (unsigned) (bufs * p.buf_cols)) p.tmem_cols *= 2;
    auto kernel = kps == 2 ? linear_fused_kernel<PAIR, SWAP, 2, KIND> : linear_fused_kernel<PAIR, SWAP, PAIR ? 2 : 1, KIND>;
    static bool configured[2][64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && (dev < 0 || dev >= 64 || !configured[kps - 1][dev])) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e == cudaSuccess && dev >= 0 && dev < 64) configured[kps - 1][dev] = true;
    }
    if (e != cudaSuccess) return 1000 + (int) e;
    CUtensorMap ma, mb;
    int rc = SWAP ? make_map(&ma, w, p.N, K, p.bn) : make_map(&ma, x, p.T, K, a_rows, ldx);
    if (rc != IIAN_OK) return rc;
    rc = SWAP ? make_map(&mb, x, p.T, K, p.x_cols, ldx) : make_map(&mb, w, p.N, K, half);
    if (rc != IIAN_OK) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned) (p.units * group));
    cfg.blockDim = dim3(LF_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    unsigned attrs = 0;
    if (group > 1) {
        attr[attrs].id = cudaLaunchAttributeClusterDimension;
        attr[attrs].val.clusterDim.x = (unsigned) group;
        attr[attrs].val.clusterDim.y = 1;
        attr[attrs++].val.clusterDim.z = 1;
    }
    if (g_iian_pdl) {
        attr[attrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[attrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    cfg.attrs = attr;
    cfg.numAttrs = attrs;
    e = cudaLaunchKernelEx(&cfg, kernel, ma, mb, (const LfArgs) p);
    return e == cudaSuccess ? IIAN_OK : 1000 + (int) e;
}

static int lf_check(int T, int N, int K, const void * x, long long ldx, const void * w, const int * status) {
    if (K <= 0 || K % 8 != 0 || ldx < K || ldx % 8 != 0 || status == nullptr) return IIAN_ERR_SHAPE;
    if (((uintptr_t) x & 15) || ((uintptr_t) w & 15)) return IIAN_ERR_ALIGN;
    if (N > 2147483647 - 512 || T > 2147483647 - 512) return IIAN_ERR_LIMIT;
    return IIAN_OK;
}

static int lf_even(int n, int parts, int step) { return std::max(32, ((n + parts - 1) / parts + step - 1) / step * step); }

// The tile and the shares of K that a call of these sizes takes: the least of an estimate in us, whose constants were fitted to 35 shapes from
// 1 x 4,096 x 1,024 to 4,096 x 1,024 x 1,024 with one block of K a stage.  Timed in every form as the stages are now, the form it takes is 2.3 %
// slower than the best one on average, and 17 % at most (256 x 4,096 x 12,288: 39.8 us, 34.1).  A K block costs the longest of its copies
// (of an SM, and of all together), its products, and the fifth of a microsecond or so that a stage's instructions and commit take (less with two
// blocks a stage: an estimate told of that chose worse); the operands come from memory; then come the epilogue of a tile and, where K is shared,
// the exchange of the parts.  Sums in float32 over a long K stay with tiles of 128 columns, which leave room for two accumulators.
static double lf_estimate(int T, int N, int K, int sms, bool pair, bool swap, int bn, int ks) {
    const int rows = pair ? 256 : 128, group = pair ? 2 : 1, a_rows = pair || T >= 128 ? 128 : (T + 7) / 8 * 8, x_cols = (T + 15) / 16 * 16;
    const double tiles = (swap ? 1.0 : (double) ((T + rows - 1) / rows)) * ((N + bn - 1) / bn), ctas = tiles * ks * group;
    int slots = sms / (group * ks) * (group * ks);
    if (ks >= 4) slots = std::min(slots, sms - sms / (ks > 4 ? 9 : 12));          // clusters of four to eight leave some SMs of a GPC over
    const double waves = (double) (long long) ((ctas + slots - 1) / slots), active = std::min(ctas, (double) slots);
    const int kb = ((K + TC_BK - 1) / TC_BK + ks - 1) / ks, per = ((bn / 4 + ks - 1) / ks) | 1;
    if (swap) {
        const double block = std::max((bn + x_cols) * 128.0 * active / 12.2e6, std::max(0.217, x_cols * 2 / 1850.0 * 1.96));
        const double work = waves * kb * block, memory = 2.0 * K * ((double) N + T) / 5.28e6;    // the shorter one is not hidden as a whole
        const double t = std::max(work, memory) + 0.25 * std::min(work, memory);
        return t + (ks == 1 ? 0.17 + 0.86 * T / 128.0 : 1.31 + waves * 4.0 * ks * x_cols * per * 16 / 131072.0);
    }
    const double fill = (a_rows + (pair ? bn / 2 : bn)) * 128.0 / std::min(131.5e3, 17.8e6 / active);
    const double t = std::max(waves * kb * std::max(fill, std::max(0.253, bn * 2 / 1850.0 * 1.5)), 2.0 * K * ((double) N + T) / 3.32e6);
    return t + (ks == 1 ? 2.74 * bn / 256 : 1.48 + waves * 10.4 * ks * a_rows * per * 16 / 131072.0);
}

// Whether w's rows are the product's: up to 64 rows of x always (1 x 4,096 x 4,096 7.8 us, the other way 8.9; 61 x 4,096 x 12,288 21.2 and 22.6; a
// row of x then costs 16 columns of a product where it cost 128 rows, and with them the power that bounds a long run of such calls), up to 128
// where K is long enough to matter (128 x 4,096 x 4,096 12.6 and 12.8, 96 x 2,048 x 8,192 11.8 and 12.0, but 100 x 4,096 x 1,024 7.3 and 6.1).
static bool lf_swaps(int T, int K) { return T <= 64 || (T <= TC_BM && K >= 2048); }

static void lf_plan(int T, int N, int K, int sms, bool out_f32, bool * pair, bool * swap, int * bn, int * ks) {
    struct Known { int T, N, K, sms, f32, pair, bn, ks; };
    static thread_local Known known[16] = {};                // by sizes alone: a model's few products come again and again
    Known & k = known[((unsigned) T * 31u + (unsigned) N * 7u + (unsigned) K) % 16u];
    *swap = lf_swaps(T, K);
    if (!(k.T == T && k.N == N && k.K == K && k.sms == sms && k.f32 == (int) out_f32 && k.bn > 0)) {
        static const int columns[] = {32, 48, 64, 96, 112, 128, 160, 192, 224, 256}, shares[] = {1, 2, 3, 4, 6};
        const int blocks = (K + TC_BK - 1) / TC_BK, most = *swap || (out_f32 && K > 6144) ? 128 : 256;
        double best = 1e300;
        for (int p = 0; p < (T > TC_BM ? 2 : 1); p++)
            for (int c : columns)
                for (int s : shares) {
                    if (c > most || (p && c % 32 != 0) || s > (p ? 4 : 6) || s > (p ? (blocks + 1) / 2 : blocks)) continue;
                    const long long ctas = (*swap ? 1LL : (long long) ((T + (p ? 255 : 127)) / (p ? 256 : 128))) * ((N + c - 1) / c) * (p ? 2 : 1);
                    if (s > 1 && ctas >= sms) break;
                    const double t = lf_estimate(T, N, K, sms, p != 0, *swap, c, s);
                    if (t < best) { best = t; k = {T, N, K, sms, (int) out_f32, p, c, s}; }
                    if (c > N) break;
                }
    }
    *pair = k.pair != 0;
    *bn = k.bn;
    *ks = k.ks;
}

}  // namespace iian

using namespace iian;

// x [T, K] bf16, rows ldx apart; w [N, K] bf16; status: two ints the host reads, as for iian_gemm_tcgen05.  form 0: chosen here; else
// pair | bn << 1 | rows << 14 | ks << 16 (rows: w's rows are the product's, bn up to 128, for x of up to 128 rows; bn a multiple of 16 from 32 to 256, on pairs of 32; 1 to 8 CTAs that share K, or 1 to 4 pairs).
IIAN_API int iian_linear_act(const void * x, long long ldx, const void * w, const float * bias, const void * residual, int res_dtype,
                             long long ldr, void * out, int out_dtype, long long ldo, int T, int N, int K, int act, int form, int * status,
                             cudaStream_t stream) {
    if (T <= 0 || N <= 0) return IIAN_OK;
    const int rc = lf_check(T, N, K, x, ldx, w, status);
    if (rc != IIAN_OK) return rc;
    LfArgs p = {};
    if (!linear_epilogue(p.epi, bias, residual, res_dtype, ldr, out, out_dtype, ldo, act)) return IIAN_ERR_DTYPE;
    const int sms = lf_sms();
    p.T = T; p.N = N;
    p.status = (TcStatus *) status;
    const int blocks = (K + TC_BK - 1) / TC_BK;
    bool pair = false, swap = false;
    if (form == 0) lf_plan(T, N, K, sms, out_dtype == IIAN_F32, &pair, &swap, &p.bn, &p.ks);
    if (form != 0) {
        pair = form & 1;
        swap = form >> 14 & 1;
        p.bn = (form >> 1) & 0x1fff;
        p.ks = form >> 16;
        if ((swap && (pair || T > TC_BM || p.bn > TC_BM)) || p.bn < 32 || p.bn > 256 || p.bn % (pair ? 32 : 16) != 0 || p.ks < 1 || p.ks > (pair ? 4 : 8) || p.ks > (pair ? (blocks + 1) / 2 : blocks) || (p.ks > 1 && p.bn / 4 < p.ks)) return IIAN_ERR_SHAPE;
    }
    const LinearEpilogue & e = p.epi;
    const bool whole = N % 4 == 0 && e.out_vec && (bias == nullptr || e.bias_vec) && (residual == nullptr || (e.res_vec && !e.res_bf16));
    auto go = [&](auto kind) {
        constexpr int KIND = decltype(kind)::value;
        return pair ? lf_launch<true, false, KIND>(p, x, ldx, w, K, sms, stream)
             : swap ? lf_launch<false, true, KIND>(p, x, ldx, w, K, sms, stream) : lf_launch<false, false, KIND>(p, x, ldx, w, K, sms, stream);
    };
    if (!whole) return go(std::integral_constant<int, LF_ANY>());
    if (residual == nullptr) return e.out_bf16 ? go(std::integral_constant<int, LF_BF16>()) : go(std::integral_constant<int, LF_F32>());
    return e.out_bf16 ? go(std::integral_constant<int, LF_BF16_RES>()) : go(std::integral_constant<int, LF_F32_RES>());
}

// Partial sums of a row (8 bytes each) that a call leaves; form as above (0: the one chosen), ks 1, any bn where w's rows are the product's.
static int lf_score_form(int T, int N, int form, bool * pair, bool * swap) {
    const int sms = lf_sms();
    *pair = T > TC_BM;
    *swap = !*pair;          // (61 rows of x behind 4,096: 213 us, x's rows as the product's 237)
    if (form != 0) {
        *pair = form & 1;
        *swap = form >> 14 & 1;
        const int bn = (form >> 1) & 0x1fff, step = *pair ? 32 : *swap ? 1 : 16;
        return (*swap && (*pair || T > TC_BM || bn > TC_BM)) || bn < 32 || bn > 256 || bn % step != 0 ? 0 : bn;
    }
    const int m_tiles = (T + (*pair ? 256 : 128) - 1) / (*pair ? 256 : 128), units = *pair ? sms / 2 : sms, most = *swap ? TC_BM : 256;
    if (*pair && m_tiles > 8) return 256;
    const long long waves = std::max<long long>(1, ((long long) m_tiles * ((N + most - 1) / most) + units - 1) / units);
    return std::min(most, lf_even(N, (int) std::min<long long>(N, waves * units / m_tiles), *pair ? 32 : *swap ? 1 : 16));
}
IIAN_API int iian_linear_logprobs_tiles(int T, int N, int form) {
    if (T <= 0 || N <= 0) return 0;
    bool pair, swap;
    const int bn = lf_score_form(T, N, form, &pair, &swap);
    return bn < 32 ? 0 : (swap ? 4 : 2) * ((N + bn - 1) / bn);
}

// targets [T]; lp, lse [T] float32; part: [tiles][T] pairs of floats, tiles as iian_linear_logprobs_tiles says.
IIAN_API int iian_linear_logprobs(const void * x, long long ldx, const void * w, const int * targets, float * lp, float * lse, float * part,
                                  int T, int N, int K, float cap, int form, int * status, cudaStream_t stream) {
    if (T <= 0) return IIAN_OK;
    if (N <= 0) return IIAN_ERR_SHAPE;
    int rc = lf_check(T, N, K, x, ldx, w, status);
    if (rc != IIAN_OK) return rc;
    if (part == nullptr || cap < 0.0f) return IIAN_ERR_SHAPE;
    LfArgs p = {};
    const int sms = lf_sms();
    bool pair, swap;
    p.T = T; p.N = N;
    p.bn = lf_score_form(T, N, form, &pair, &swap);
    p.ks = 1;
    if (p.bn < 32) return IIAN_ERR_SHAPE;
    p.status = (TcStatus *) status;
    p.score = {(float2 *) part, targets, lp, cap};
    rc = pair ? lf_launch<true, false, LF_SCORE>(p, x, ldx, w, K, sms, stream)
       : swap ? lf_launch<false, true, LF_SCORE>(p, x, ldx, w, K, sms, stream) : lf_launch<false, false, LF_SCORE>(p, x, ldx, w, K, sms, stream);
    if (rc != IIAN_OK) return rc;
    return lf_join(part, (swap ? 4 : 2) * ((N + p.bn - 1) / p.bn), T, N, targets, lp, lse, stream);
}

// The same from logits in memory, a piece of the vocabulary at a time: logits [T, P] float32 hold columns v0 .. v0 + P; every `columns` of them
// become one of part[first ..] (the last piece's call is followed by one of iian_linear_logprobs_join over all parts).
IIAN_API int iian_linear_logprobs_piece(const float * logits, int T, int P, int v0, const int * targets, float * lp, float * part, int first,
                                        int columns, float cap, cudaStream_t stream) {
    if (T <= 0 || P <= 0) return IIAN_OK;
    if (columns <= 0 || P > 2147483647 - columns || (P + columns - 1) / columns > 65535 || first < 0 || cap < 0.0f) return IIAN_ERR_SHAPE;
    return iian_launch(logprobs_piece_kernel, dim3((unsigned) T, (unsigned) ((P + columns - 1) / columns)), dim3(256), 0, stream, logits, T, P, v0, targets, lp,
                       (float2 *) part, first, columns, cap);
}
IIAN_API int iian_linear_logprobs_join(const float * part, int parts, int T, int V, const int * targets, float * lp, float * lse, cudaStream_t stream) {
    if (T <= 0) return IIAN_OK;
    if (parts <= 0) return IIAN_ERR_SHAPE;
    return lf_join(part, parts, T, V, targets, lp, lse, stream);
}
