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
// Few rows of x: a stage holds only the rows there are (in eights), so that nearly all of shared memory is weights on their way.  The
// product then still reads 128 rows of shared memory; what lies behind the real ones only reaches rows of the accumulator that nobody
// reads.
//
// Few tiles: the K blocks of a tile are shared by a cluster of `ks` CTAs.  Each leaves its part in its shared memory, and each adds up all
// parts, in their order, for its share of the tile.
//
// The softmax's sums: a thread walks its row's columns with a running maximum and sum and leaves them per tile; a second kernel joins a
// row's.  The maximum is the running one, so no exponential overflows; an empty sum has the maximum minus infinity.
//
// Every wait is bounded, as in gemm_tcgen05.cu; a producer that gives up waits, bounded too, for the copies it still has under way.
#include <math_constants.h>

#include <algorithm>

#include "common.cuh"
#include "epilogue.cuh"
#include "tc_product.cuh"

namespace iian {

constexpr int LF_STAGES = 16;             // barriers there are; how many are used follows from the size of a stage
constexpr float kLog2e = 1.4426950408889634f;

struct LfScore {
    float2 * part;                        // [column tiles][T]: maximum and sum of a row's columns in a tile
    const int * targets;
    float * lp;                           // receives the target's logit
    float cap;                            // 0: none
};

struct LfArgs {
    int T, N, K, bn, ks, stages, a_rows, stage_bytes;
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
// c tanh(z / c) with the hardware's exponential: tanh's absolute error is a few 1e-7
__device__ __forceinline__ float lf_cap_fast(float z, float cap, float two_over_cap_log2e) {
    return cap * (1.0f - __fdividef(2.0f, 1.0f + lf_exp2(z * two_over_cap_log2e)));
}

// 32 columns of a row, `live` of them in the matrix, into the row's running maximum and sum
__device__ __forceinline__ void lf_take(const unsigned * r, int live, float cap, float two_over_cap_log2e, float & m, float & s) {
    float z[32], mx[4] = {-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
    for (int i = 0; i < 32; i++) {
        z[i] = __uint_as_float(r[i]);
        if (cap != 0.0f) z[i] = lf_cap_fast(z[i], cap, two_over_cap_log2e);
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

template <bool PAIR, bool SCORE>
__global__ void __launch_bounds__(TC_THREADS, 1) linear_fused_kernel(const __grid_constant__ CUtensorMap map_a,
                                                                     const __grid_constant__ CUtensorMap map_b, const LfArgs p) {
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char * smem = (unsigned char *) (((uintptr_t) smem_raw + 1023) & ~(uintptr_t) 1023);
    constexpr int KPS = PAIR ? 2 : 1;     // blocks of K a stage
    constexpr int ROWS = PAIR ? 2 * TC_BM : TC_BM;
    __shared__ __align__(8) unsigned long long full_bar[LF_STAGES], empty_bar[LF_STAGES], acc_full[2], acc_empty[2];
    __shared__ unsigned tmem_base_s;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int bn = p.bn, half = PAIR ? bn / 2 : bn, stages = p.stages;
    const unsigned cluster_rank = PAIR || p.ks > 1 ? cluster_cta_rank() : 0u;
    const unsigned rank = PAIR ? cluster_rank : 0u;                           // which CTA of a pair
    const int group = PAIR ? 2 : p.ks, unit = (int) blockIdx.x / group, units = (int) gridDim.x / group;
    const int a_bytes = p.a_rows * TC_BK * 2, b_bytes = half * TC_BK * 2, kb_bytes = a_bytes + b_bytes;
    const int blocks = (p.K + TC_BK - 1) / TC_BK, all_kb = (blocks + KPS - 1) / KPS;
    const int kb0 = PAIR ? 0 : (int) ((long long) all_kb * cluster_rank / p.ks);
    const int kb1 = PAIR ? all_kb : (int) ((long long) all_kb * (cluster_rank + 1) / p.ks);
    const int m_tiles = (p.T + ROWS - 1) / ROWS, n_tiles = (p.N + bn - 1) / bn;
    const long long num_tiles = (long long) m_tiles * n_tiles;
    const int acc_cols = (bn + 31) & ~31;
    unsigned tmem_cols = 64;
    while (tmem_cols < 2u * acc_cols) tmem_cols *= 2;

    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; s++) { mbar_init(smem_addr(&full_bar[s]), 1); mbar_init(smem_addr(&empty_bar[s]), 1); }
        for (int b = 0; b < 2; b++) { mbar_init(smem_addr(&acc_full[b]), 1); mbar_init(smem_addr(&acc_empty[b]), PAIR ? 8 : 4); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        if constexpr (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_base_s)), "r"(tmem_cols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_base_s)), "r"(tmem_cols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (PAIR) cluster_sync_all();       // the peer's barriers exist before anything arrives on them
    tc_fence_after();
    const unsigned tmem_base = tmem_base_s;

    if (warp == 0 && lane == 0) {
        // ---- producer ---------------------------------------------------------------------------------------
        int it = 0;
        bool gave_up = false;
        for (long long tile = unit; tile < num_tiles && !gave_up; tile += units) {
            const int m0 = (int) (tile % m_tiles) * ROWS + (int) rank * TC_BM, n0 = (int) (tile / m_tiles) * bn + (int) rank * half;
            for (int kb = kb0; kb < kb1; kb++, it++) {
                const int s = it % stages;
                if (!mbar_wait(smem_addr(&empty_bar[s]), ((it / stages) & 1) ^ 1)) { p.status->code = 1; p.status->where = it; gave_up = true; break; }
                const unsigned to = smem_addr(smem + s * p.stage_bytes);
                if constexpr (PAIR) {
                    const unsigned bar = map_to_cta(smem_addr(&full_bar[s]), 0);
                    if (rank == 0) mbar_expect_tx(smem_addr(&full_bar[s]), 2 * KPS * kb_bytes);
#pragma unroll
                    for (int j = 0; j < KPS; j++) {
                        tma_load_2d_pair(to + j * kb_bytes, &map_a, (kb * KPS + j) * TC_BK, m0, bar);
                        tma_load_2d_pair(to + j * kb_bytes + a_bytes, &map_b, (kb * KPS + j) * TC_BK, n0, bar);
                    }
                } else {
                    const unsigned bar = smem_addr(&full_bar[s]);
                    mbar_expect_tx(bar, kb_bytes);
                    tma_load_2d(to, &map_a, kb * TC_BK, m0, bar);
                    tma_load_2d(to + a_bytes, &map_b, kb * TC_BK, n0, bar);
                }
            }
        }
        if (gave_up) {                            // its copies land before the CTA may leave
            if (rank == 0)
                for (int i = max(0, it - stages); i < it; i++) mbar_wait(smem_addr(&full_bar[i % stages]), (i / stages) & 1);
        } else if (PAIR) {                        // the last commits still arrive on this CTA's barriers
            for (int i = 0; i < stages; i++, it++)
                if (!mbar_wait(smem_addr(&empty_bar[it % stages]), ((it / stages) & 1) ^ 1)) { p.status->code = 5; p.status->where = it; break; }
        }
    } else if (warp == 1 && lane == 0 && rank == 0) {
        // ---- MMA issuer -------------------------------------------------------------------------------------
        const unsigned idesc = instr_desc_bf16(ROWS, bn);
        int it = 0, use = 0;
        bool gave_up = false;
        for (long long tile = unit; tile < num_tiles && !gave_up; tile += units, use++) {
            const int buf = use & 1;
            if (!mbar_wait(smem_addr(&acc_empty[buf]), ((use >> 1) & 1) ^ 1)) { p.status->code = 4; p.status->where = use; break; }
            tc_fence_after();
            const unsigned d_tmem = tmem_base + (unsigned) (buf * acc_cols);
            for (int kb = kb0; kb < kb1; kb++, it++) {
                const int s = it % stages;
                if (!mbar_wait(smem_addr(&full_bar[s]), (it / stages) & 1)) { p.status->code = 2; p.status->where = it; gave_up = true; break; }
                tc_fence_after();
#pragma unroll
                for (int j = 0; j < KPS; j++) {
                    const unsigned long long da = smem_desc_sw128(smem_addr(smem + s * p.stage_bytes + j * kb_bytes));
                    const unsigned long long db = smem_desc_sw128(smem_addr(smem + s * p.stage_bytes + j * kb_bytes + a_bytes));
#pragma unroll
                    for (int k = 0; k < TC_BK / 16; k++) {
                        const unsigned acc = kb > kb0 || j > 0 || k > 0 ? 1u : 0u;
                        if constexpr (PAIR) tc_mma_pair(d_tmem, da + (unsigned long long) (k * 2), db + (unsigned long long) (k * 2), idesc, acc);
                        else tc_mma(d_tmem, da + (unsigned long long) (k * 2), db + (unsigned long long) (k * 2), idesc, acc);
                    }
                }
                if constexpr (PAIR) tc_commit_pair(smem_addr(&empty_bar[s]));
                else tc_commit(smem_addr(&empty_bar[s]));
            }
            if (!gave_up) {
                if constexpr (PAIR) tc_commit_pair(smem_addr(&acc_full[buf]));
                else tc_commit(smem_addr(&acc_full[buf]));
            }
        }
    } else if (warp >= 2) {
        // ---- epilogue: warp w reads tensor-memory lanes 32 * (w % 4) .. + 31 -----------------------------------
        const int q = warp & 3;
        const float cap_factor = SCORE && p.score.cap != 0.0f ? 2.0f * kLog2e / p.score.cap : 0.0f;
        int use = 0;
        for (long long tile = unit; tile < num_tiles; tile += units, use++) {
            const int buf = use & 1;
            const int n_tile = (int) (tile / m_tiles), m0 = (int) (tile % m_tiles) * ROWS + (int) rank * TC_BM, n0 = n_tile * bn;
            if (!mbar_wait(smem_addr(&acc_full[buf]), (use >> 1) & 1)) {
                if (lane == 0) { p.status->code = 3; p.status->where = use; }
                break;
            }
            tc_fence_after();
            const int row = m0 + q * 32 + lane, cols = min(bn, p.N - n0);
            const unsigned acc = tmem_base + ((unsigned) (q * 32) << 16) + (unsigned) (buf * acc_cols);
            if (m0 + q * 32 < p.T) {              // (a warp whose rows are all behind the last one has nothing to do)
                if constexpr (SCORE) {
                    float m = -CUDART_INF_F, s = 0.0f;
                    const int wanted = row < p.T ? p.score.targets[row] : -1, target = wanted < 0 ? -1 : wanted - n0;
#pragma unroll 1
                    for (int c0 = 0; c0 < cols; c0 += 32) {
                        unsigned r[32];
                        tc_ld32(acc + (unsigned) c0, r);
                        tc_wait_ld();
                        lf_take(r, cols - c0, p.score.cap, cap_factor, m, s);
                        if (target >= c0 && target < c0 + 32 && target < cols) {
                            const float z = __uint_as_float(lf_pick(r, target - c0));
                            p.score.lp[row] = p.score.cap != 0.0f ? p.score.cap * tanhf(z / p.score.cap) : z;
                        }
                    }
                    if (row < p.T) p.score.part[(size_t) n_tile * p.T + row] = make_float2(m, s);
                } else if (PAIR || p.ks == 1) {
#pragma unroll 1
                    for (int c0 = 0; c0 < cols; c0 += 32) {
                        unsigned r[32];
                        tc_ld32(acc + (unsigned) c0, r);
                        tc_wait_ld();
                        if (row < p.T) {
#pragma unroll
                            for (int v = 0; v < 4; v++) {
                                const int live = cols - c0 - 8 * v;
                                if (live > 0) {
                                    float y[8];
#pragma unroll
                                    for (int i = 0; i < 8; i++) y[i] = __uint_as_float(r[8 * v + i]);
                                    p.epi.store8(y, row, n0 + c0 + 8 * v, live);
                                }
                            }
                        }
                    }
                } else {
                    // this CTA's part of the sums, for the cluster: rows of bn + 4 floats over the ring, whose copies and products are all done
                    float * part = reinterpret_cast<float *>(smem) + (size_t) (q * 32 + lane) * (bn + 4);
#pragma unroll 1
                    for (int c0 = 0; c0 < bn; c0 += 32) {
                        unsigned r[32];
                        tc_ld32(acc + (unsigned) c0, r);
                        tc_wait_ld();
                        if (row < p.T) {
#pragma unroll
                            for (int v = 0; v < 8; v++)
                                if (c0 + 4 * v < bn) *reinterpret_cast<uint4 *>(part + c0 + 4 * v) = make_uint4(r[4 * v], r[4 * v + 1], r[4 * v + 2], r[4 * v + 3]);
                        }
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if constexpr (PAIR) mbar_arrive_cluster(map_to_cta(smem_addr(&acc_empty[buf]), 0));
                else mbar_arrive(smem_addr(&acc_empty[buf]));
            }
        }
    }
    // ---- common exit: everybody arrives here, also after a wait that gave up -----------------------------------
    tc_fence_before();
    __syncthreads();
    __syncwarp();
    if constexpr (!PAIR && !SCORE) {
        if (p.ks > 1) {
            cluster_sync_all();                   // all parts lie ready
            const int m0 = (unit % m_tiles) * ROWS, n0 = (unit / m_tiles) * bn;
            const int rows = min(TC_BM, p.T - m0), cols = min(bn, p.N - n0), per_row = (cols + 7) / 8;
            const int pieces = rows * per_row, from = (int) ((long long) pieces * cluster_rank / p.ks), to = (int) ((long long) pieces * (cluster_rank + 1) / p.ks);
            const unsigned base = smem_addr(smem);
            for (int i = from + (int) threadIdx.x; i < to; i += TC_THREADS) {
                const int row = i / per_row, c = (i - row * per_row) * 8;
                const unsigned at = base + (unsigned) (row * (bn + 4) + c) * 4u;
                float y[8];
#pragma unroll
                for (int j = 0; j < 8; j++) y[j] = 0.0f;
#pragma unroll 4
                for (int r = 0; r < p.ks; r++) {
                    const unsigned peer = map_to_cta(at, (unsigned) r);
                    float a[8];
                    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(a[0]), "=f"(a[1]), "=f"(a[2]), "=f"(a[3]) : "r"(peer) : "memory");
                    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(a[4]), "=f"(a[5]), "=f"(a[6]), "=f"(a[7]) : "r"(peer + 16) : "memory");
#pragma unroll
                    for (int j = 0; j < 8; j++) y[j] += a[j];
                }
                p.epi.store8(y, (size_t) (m0 + row), n0 + c, cols - c);
            }
            __syncwarp();
            cluster_sync_all();                   // nobody leaves while its part is read
        }
    }
    if constexpr (PAIR) cluster_sync_all();
    if (warp == 1) {
        tc_fence_after();
        if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(tmem_cols) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(tmem_cols) : "memory");
    }
}

// A row's maxima and sums of all column tiles become its log-sum-exp, the target's logit its log-probability.  A CTA has `rows` rows (a
// power of two up to 32) and 512 / rows threads for each.  A target below 0 is none: 0; one beyond the vocabulary is no number.
__global__ void __launch_bounds__(512) logprobs_join_kernel(const float2 * __restrict__ part, int n_tiles, int T, int V, int rows,
                                                            const int * __restrict__ targets, float * __restrict__ lp, float * __restrict__ lse) {
    __shared__ float sm[512], ss[512];
    const int r = threadIdx.x & (rows - 1), seg = threadIdx.x / rows, segs = 512 / rows;
    const long long row = (long long) blockIdx.x * rows + r;
    float m = -CUDART_INF_F, s = 0.0f;
    auto add = [&](float m2, float s2) {
        const float m1 = fmaxf(m, m2), ref = lf_finite_or_zero(m1) * kLog2e;
        s = (s == 0.0f ? 0.0f : s * lf_exp2(fmaf(m, kLog2e, -ref))) + (s2 == 0.0f ? 0.0f : s2 * lf_exp2(fmaf(m2, kLog2e, -ref)));
        m = m1;
    };
    if (row < T) {
#pragma unroll 4
        for (int i = seg; i < n_tiles; i += segs) {
            const float2 v = part[(size_t) i * T + row];
            add(v.x, v.y);
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

// Columns v0 .. v0 + P of the logits of T rows, as they lie in memory, into the rows' maxima and sums: part `split` of gridDim.y of a piece
// whose parts begin at part[first].  For element types and sizes that the tensor cores' product does not take.
__global__ void __launch_bounds__(256) logprobs_piece_kernel(const float * __restrict__ logits, int T, int P, int v0, const int * __restrict__ targets,
                                                             float * __restrict__ lp, float2 * __restrict__ part, int first, float cap) {
    __shared__ float sm[8], ss[8];
    const size_t row = blockIdx.x;
    const int splits = gridDim.y, c0 = (int) ((long long) P * blockIdx.y / splits), c1 = (int) ((long long) P * (blockIdx.y + 1) / splits);
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
    int rows = 1;
    while (rows < 32 && rows < T) rows *= 2;
    logprobs_join_kernel<<<(unsigned) ((T + rows - 1) / rows), 512, 0, stream>>>((const float2 *) part, n_tiles, T, V, rows, targets, lp, lse);
    return iian_launch_status();
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

// bn, ks as given; pair: tiles of 256 rows on pairs of SMs.
template <bool PAIR, bool SCORE>
static int lf_launch(LfArgs & p, const void * x, long long ldx, const void * w, int sms, cudaStream_t stream) {
    constexpr int KPS = PAIR ? 2 : 1, ROWS = PAIR ? 2 * TC_BM : TC_BM;
    // All of it whatever the call needs: two CTAs of a cluster that each waited for the tensor memory of an SM's other CTA, those two in turn
    // waiting for their clusters, would never end, so no SM may hold two.
    constexpr int kRing = 208 * 1024, smem = kRing + 1024;
    p.a_rows = PAIR || p.T >= TC_BM ? TC_BM : (p.T + 7) / 8 * 8;
    const int half = PAIR ? p.bn / 2 : p.bn;
    p.stage_bytes = KPS * (p.a_rows + half) * TC_BK * 2;
    const int over = (TC_BM - p.a_rows) * TC_BK * 2;                   // the last stage's product reads 128 rows too
    p.stages = std::min(LF_STAGES, (kRing - over) / p.stage_bytes);
    static_assert(TC_BM * (256 + 4) * 4 <= kRing, "a tile's sums fit the ring");
    auto kernel = linear_fused_kernel<PAIR, SCORE>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return 1000 + (int) e;
    CUtensorMap ma, mb;
    int rc = make_map(&ma, x, p.T, p.K, p.a_rows, ldx);
    if (rc != IIAN_OK) return rc;
    rc = make_map(&mb, w, p.N, p.K, half);
    if (rc != IIAN_OK) return rc;
    const long long tiles = (long long) ((p.T + ROWS - 1) / ROWS) * ((p.N + p.bn - 1) / p.bn);
    const int group = PAIR ? 2 : p.ks;
    const long long units = p.ks > 1 ? tiles : std::min<long long>(tiles, sms / group);
    if (units * group > 2147483647LL) return IIAN_ERR_LIMIT;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned) (units * group));
    cfg.blockDim = dim3(TC_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned) group;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = group > 1 ? 1 : 0;
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

}  // namespace iian

using namespace iian;

// x [T, K] bf16, rows ldx apart; w [N, K] bf16; status: two ints the host reads, as for iian_gemm_tcgen05.  form 0: chosen here; else
// pair | bn << 1 | ks << 16 (a multiple of 16 from 32 to 256, on pairs of 32; 1 to 8 CTAs that share K, 1 on pairs).
IIAN_API int iian_linear_act(const void * x, long long ldx, const void * w, const float * bias, const void * residual, int res_dtype,
                             long long ldr, void * out, int out_dtype, long long ldo, int T, int N, int K, int act, int form, int * status,
                             cudaStream_t stream) {
    if (T <= 0 || N <= 0) return IIAN_OK;
    const int rc = lf_check(T, N, K, x, ldx, w, status);
    if (rc != IIAN_OK) return rc;
    LfArgs p = {};
    if (!linear_epilogue(p.epi, bias, residual, res_dtype, ldr, out, out_dtype, ldo, act)) return IIAN_ERR_DTYPE;
    const int sms = lf_sms();
    p.T = T; p.N = N; p.K = K;
    p.status = (TcStatus *) status;
    const int blocks = (K + TC_BK - 1) / TC_BK;
    bool pair = T > TC_BM;
    p.bn = pair ? 256 : lf_even(N, (N + 127) / 128, 16);
    p.ks = 1;
    if (!pair) {
        const int tiles = (N + p.bn - 1) / p.bn;
        while (p.ks < 8 && tiles * p.ks * 2 <= sms && blocks >= p.ks * 4) p.ks *= 2;
    }
    if (form != 0) {
        pair = form & 1;
        p.bn = (form >> 1) & 0x7fff;
        p.ks = form >> 16;
        if (p.bn < 32 || p.bn > 256 || p.bn % (pair ? 32 : 16) != 0 || p.ks < 1 || p.ks > (pair ? 1 : 8) || p.ks > blocks) return IIAN_ERR_SHAPE;
    }
    return pair ? lf_launch<true, false>(p, x, ldx, w, sms, stream) : lf_launch<false, false>(p, x, ldx, w, sms, stream);
}

// Column tiles of a call, whose partial sums take 8 bytes a tile and row; form as above (0: the one chosen), ks 1.
static int lf_score_form(int T, int N, int form, bool * pair) {
    const int sms = lf_sms();
    *pair = T > TC_BM;
    if (form != 0) {
        *pair = form & 1;
        return (form >> 1) & 0x7fff;
    }
    const int m_tiles = (T + (*pair ? 256 : 128) - 1) / (*pair ? 256 : 128), units = *pair ? sms / 2 : sms;
    if (*pair && m_tiles > 8) return 256;
    const long long waves = std::max<long long>(1, ((long long) m_tiles * ((N + 255) / 256) + units - 1) / units);
    return std::min(256, lf_even(N, (int) std::min<long long>(N, waves * units / m_tiles), *pair ? 32 : 16));
}
IIAN_API int iian_linear_logprobs_tiles(int T, int N, int form) {
    if (T <= 0 || N <= 0) return 0;
    bool pair;
    const int bn = lf_score_form(T, N, form, &pair);
    return bn < 32 ? 0 : (N + bn - 1) / bn;
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
    bool pair;
    p.T = T; p.N = N; p.K = K;
    p.bn = lf_score_form(T, N, form, &pair);
    p.ks = 1;
    if (p.bn < 32 || p.bn > 256 || p.bn % (pair ? 32 : 16) != 0) return IIAN_ERR_SHAPE;
    p.status = (TcStatus *) status;
    p.score = {(float2 *) part, targets, lp, cap};
    rc = pair ? lf_launch<true, true>(p, x, ldx, w, sms, stream) : lf_launch<false, true>(p, x, ldx, w, sms, stream);
    if (rc != IIAN_OK) return rc;
    return lf_join(part, (N + p.bn - 1) / p.bn, T, N, targets, lp, lse, stream);
}

// The same from logits in memory, a piece of the vocabulary at a time: logits [T, P] float32 hold columns v0 .. v0 + P, whose `splits` parts
// become part[first ..] (the last piece's call is followed by one of iian_linear_logprobs_join over all parts).
IIAN_API int iian_linear_logprobs_piece(const float * logits, int T, int P, int v0, const int * targets, float * lp, float * part, int first,
                                        int splits, float cap, cudaStream_t stream) {
    if (T <= 0 || P <= 0) return IIAN_OK;
    if (splits <= 0 || splits > 65535 || first < 0 || cap < 0.0f) return IIAN_ERR_SHAPE;
    logprobs_piece_kernel<<<dim3((unsigned) T, (unsigned) splits), 256, 0, stream>>>(logits, T, P, v0, targets, lp, (float2 *) part, first, cap);
    return iian_launch_status();
}
IIAN_API int iian_linear_logprobs_join(const float * part, int parts, int T, int V, const int * targets, float * lp, float * lse, cudaStream_t stream) {
    if (T <= 0) return IIAN_OK;
    if (parts <= 0) return IIAN_ERR_SHAPE;
    return lf_join(part, parts, T, V, targets, lp, lse, stream);
}
