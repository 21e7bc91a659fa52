// Which experts a token takes where experts come in groups, and what they weigh.
//
//   s = sigmoid(z)  or  softmax(z) over all E outputs of the router;   c = s + correction
//   a group is E / G neighbouring outputs; its score is the sum of its `group_top` (1 or 2) largest c
//   of the `top_groups` groups with the largest scores (ties: the lower group) the `top` outputs with the largest c (ties: the lower index)
//   w = s, without the correction; with `renorm` divided by the sum of the chosen s; times `scale`
//
// Scores are formed and compared in 64 bits: which of two neighbouring scores is the larger is a whole number, and the rounding of a
// 32-bit exponential would decide it.  A score that is no number is the smallest; a row whose chosen scores are all 0 weighs 0
// (a softmax over logits of minus infinity alone is such a row).
#include "common.cuh"

namespace iian {

constexpr int kGroupsMost = 32, kGroupTopMost = 32, kGroupOutputsMost = 1024;

__device__ __forceinline__ double shfl_xor_f64(double v, int o) { return __shfl_xor_sync(0xffffffffu, v, o); }

// The order of doubles as the order of unsigned numbers: 0 is below all of them.
__device__ __forceinline__ unsigned long long order_key(double v) {
    const long long b = __double_as_longlong(v);
    return (unsigned long long) (b ^ ((b >> 63) | (long long) 0x8000000000000000ull));
}

// One warp a token.  Every group has `lanes` = 32 / (groups, rounded up to a power of two) lanes of its own, output g * per + sub + lanes * i
// lies in slot i of lane g * lanes + sub: a group's best two are a reduction over its own lanes, and a group's rank among the groups is
// a count.  The choice is a chain of `top` reductions over the warp; lane k keeps choice k.
template <int SLOTS>
__global__ void __launch_bounds__(128) moe_route_grouped_kernel(const float * __restrict__ logits, long long ld,
                                                                const float * __restrict__ correction, int E, int groups, int lanes,
                                                                int top_groups, int group_top, int top, int softmax, int renorm,
                                                                double scale, int * __restrict__ ids, float * __restrict__ wts, int N) {
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const long long t = (long long) blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (t >= N) return;
    const int per = E / groups, group = lane / lanes, sub = lane - group * lanes, first = group * per;
    const bool live = group < groups;
    const float * z = logits + t * ld;
    double s[SLOTS];
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < SLOTS; i++) {
        const int j = sub + lanes * i;
        const float v = live && j < per ? z[first + j] : -INFINITY;
        s[i] = v;
        mx = fmaxf(mx, v);
    }
    if (softmax) {
        mx = warp_max(mx);
        if (mx == -INFINITY) mx = 0.0f;                      // nothing but minus infinity: every score 0
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < SLOTS; i++) {
            s[i] = exp(s[i] - (double) mx);
            sum += s[i];
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += shfl_xor_f64(sum, o);
        const double inv = sum > 0.0 ? 1.0 / sum : (sum == 0.0 ? 0.0 : sum);
#pragma unroll
        for (int i = 0; i < SLOTS; i++) s[i] *= inv;
    } else {
#pragma unroll
        for (int i = 0; i < SLOTS; i++) s[i] = 1.0 / (1.0 + exp(-s[i]));
    }
    unsigned long long key[SLOTS];                           // 0: not to be chosen (none there, a group that is shut, taken)
    double b1 = -INFINITY, b2 = -INFINITY;                   // this lane's two largest c
#pragma unroll
    for (int i = 0; i < SLOTS; i++) {
        const int j = sub + lanes * i;
        key[i] = 0;
        if (live && j < per) {
            double c = correction != nullptr ? s[i] + (double) correction[first + j] : s[i];
            if (c != c) c = -INFINITY;
            c += 0.0;                                        // minus zero is zero
            key[i] = order_key(c);
            b2 = fmax(b2, fmin(b1, c));
            b1 = fmax(b1, c);
        }
    }
    if (top_groups < groups) {
        for (int o = 1; o < lanes; o <<= 1) {
            const double o1 = shfl_xor_f64(b1, o), o2 = shfl_xor_f64(b2, o);
            b2 = fmax(fmax(b2, o2), fmin(b1, o1));
            b1 = fmax(b1, o1);
        }
        double gs = group_top == 2 && per > 1 ? b1 + b2 : b1;
        if (gs != gs) gs = -INFINITY;
        int ahead = 0;                                       // groups that come before this lane's
        for (int g = 0; g < groups; g++) {
            const double other = __shfl_sync(0xffffffffu, gs, g * lanes);
            ahead += other > gs || (other == gs && g < group);
        }
        if (ahead >= top_groups) {
#pragma unroll
            for (int i = 0; i < SLOTS; i++) key[i] = 0;
        }
    }
    double mine = 0.0;                                       // choice `lane`
    int mine_e = 0;
    unsigned long long best = 0;
    int at = 0;
    auto look = [&]() {
        best = 0;
        at = 0;
#pragma unroll
        for (int i = 0; i < SLOTS; i++)
            if (key[i] > best) { best = key[i]; at = i; }    // (a lane's outputs rise: ties keep the lower)
    };
    look();
    for (int k = 0; k < top; k++) {
        const unsigned hi = (unsigned) (best >> 32), most = __reduce_max_sync(0xffffffffu, hi);
        const unsigned lo = hi == most ? (unsigned) best : 0u, most_lo = __reduce_max_sync(0xffffffffu, lo);
        const bool ties = hi == most && lo == most_lo;
        const int e = ties ? first + sub + lanes * at : 0x7fffffff;
        const int won = __reduce_min_sync(0xffffffffu, e);
        const int from = __ffs(__ballot_sync(0xffffffffu, e == won)) - 1;
        double sc = 0.0;
        if (e == won) {
#pragma unroll
            for (int i = 0; i < SLOTS; i++)
                if (i == at) { sc = s[i]; key[i] = 0; }
            look();
        }
        sc = __shfl_sync(0xffffffffu, sc, from);
        if (lane == k) { mine = sc; mine_e = won; }
    }
    if (renorm) {
        double sum = lane < top ? mine : 0.0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += shfl_xor_f64(sum, o);
        mine = sum == 0.0 ? 0.0 : mine / sum;
    }
    if (lane < top) {
        ids[t * top + lane] = mine_e;
        wts[t * top + lane] = (float) (mine * scale);
    }
}

}  // namespace iian

using namespace iian;

// logits [N, E] float32, rows `ld` apart; correction [E] float32 or null; ids / wts [N, top].  softmax: 0 sigmoid, 1 softmax.
IIAN_API int iian_moe_route_grouped(const float * logits, long long ld, const float * correction, int E, int groups, int top_groups,
                                    int group_top, int top, int softmax, int renorm, float scale, int * ids, float * wts, int N,
                                    cudaStream_t stream) {
    if (N <= 0) return IIAN_OK;
    if (E <= 0 || groups <= 0 || E % groups != 0 || top_groups <= 0 || top_groups > groups || (group_top != 1 && group_top != 2)) return IIAN_ERR_SHAPE;
    if (top <= 0 || top > top_groups * (E / groups)) return IIAN_ERR_SHAPE;
    if (E > kGroupOutputsMost || groups > kGroupsMost || top > kGroupTopMost) return IIAN_ERR_LIMIT;
    int wide = 1;
    while (wide < groups) wide *= 2;
    const int lanes = 32 / wide, slots = (E / groups + lanes - 1) / lanes, warps = 4;
    const dim3 grid((unsigned) (((long long) N + warps - 1) / warps));
    auto go = [&](auto kernel) {
        return iian_launch(kernel, grid, dim3(warps * 32), 0, stream, logits, ld, correction, E, groups, lanes, top_groups, group_top, top,
                           softmax, renorm, (double) scale, ids, wts, N);
    };
    if (slots <= 2) return go(moe_route_grouped_kernel<2>);
    if (slots <= 4) return go(moe_route_grouped_kernel<4>);
    if (slots <= 8) return go(moe_route_grouped_kernel<8>);
    if (slots <= 16) return go(moe_route_grouped_kernel<16>);
    if (slots <= 32) return go(moe_route_grouped_kernel<32>);
    return go(moe_route_grouped_kernel<64>);                 // 17 groups of 60: half of the lanes hold nothing
}
