// Which experts a token takes where experts come in groups, and what they weigh.
//
//   s = sigmoid(z)  or  softmax(z) over all E outputs of the router;   c = s + correction
//   a group is E / G neighbouring outputs; its score is the sum of its `group_top` (1 or 2) largest c
//   of the `top_groups` groups with the largest scores (ties: the lower group) the `top` outputs with the largest c (ties: the lower index)
//   w = s, without the correction; with `renorm` divided by the sum of the chosen s; times `scale`
//
// Which of two scores is the larger is a whole number, and the rounding of a 32-bit exponential would decide it where they are neighbours.  So
// the order is that of the scores in 64 bits: a warp forms them in 32, and where two scores whose order matters are nearer to one another
// than these can tell, does its token again in 64.  A score that is no number is the smallest; a row whose chosen scores are all 0
// weighs 0 (a softmax over logits of minus infinity alone is such a row).
//
// What bounds it: latency.  A token is a chain of `top` + 2 reductions and the groups' ranks, some 40 dependent shuffles, on one warp; 64 registers
// let an SM hold 32 of them, so that 8,192 tokens are 1.7 waves, and the issue slots are half full (52 %).  Sigmoid scores with a correction, 8 of
// 256 experts in 8 groups: 61 tokens 3.2 us (2.3 of them the launch), 512 3.8, 2,047 6.0, 8,192 10.8 (8.9 MB: 0.8 TB/s); every score in
// 64 bits 24 us, neighbours left to route_exact 14.5.
#include "common.cuh"

namespace iian {

constexpr int kGroupsMost = 32, kGroupTopMost = 32, kGroupOutputsMost = 1024;

__device__ __forceinline__ double shfl_xor_f64(double v, int o) { return __shfl_xor_sync(0xffffffffu, v, o); }

// The order of doubles as the order of unsigned numbers: 0 is below all of them.
__device__ __forceinline__ unsigned long long order_key(double v) {
    const long long b = __double_as_longlong(v);
    return (unsigned long long) (b ^ ((b >> 63) | (long long) 0x8000000000000000ull));
}

__device__ __forceinline__ unsigned order_key(float v) {
    const int b = __float_as_int(v);
    return (unsigned) (b ^ ((b >> 31) | (int) 0x80000000u));
}

__device__ __forceinline__ float route_sigmoid(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(1.0f + __expf(-x)));
    return y;
}

struct RouteArgs {
    const float * logits;
    long long ld;
    const float * correction;
    int E, groups, lanes, chunk, top_groups, group_top, top, softmax, renorm;
    double scale;
    int * ids;
    float * wts;
};

// One warp a token.  Every group has `lanes` = 32 / (groups, rounded up to a power of two) lanes of its own, each with `chunk` neighbouring
// outputs: a group's best two are a reduction over its own lanes, and a group's rank among the groups is a count.  The choice is a
// chain of `top` reductions over the warp; lane k keeps choice k.
template <int SLOTS>
__device__ __noinline__ void route_exact(const RouteArgs & p, long long t) {
    const int lane = threadIdx.x & 31, per = p.E / p.groups, group = lane / p.lanes, j0 = (lane - group * p.lanes) * p.chunk;
    const int first = group * per + j0, held = group < p.groups ? max(0, min(p.chunk, per - j0)) : 0;
    const float * z = p.logits + t * p.ld + first;
    double s[SLOTS];
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < SLOTS; i++) {
        const float v = i < held ? z[i] : -INFINITY;
        s[i] = v;
        mx = fmaxf(mx, v);
    }
    if (p.softmax) {
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
        key[i] = 0;
        if (i < held) {
            double c = p.correction != nullptr ? s[i] + (double) p.correction[first + i] : s[i];
            if (c != c) c = -INFINITY;
            c += 0.0;                                        // minus zero is zero
            key[i] = order_key(c);
            b2 = fmax(b2, fmin(b1, c));
            b1 = fmax(b1, c);
        }
    }
    if (p.top_groups < p.groups) {
        for (int o = 1; o < p.lanes; o <<= 1) {
            const double o1 = shfl_xor_f64(b1, o), o2 = shfl_xor_f64(b2, o);
            b2 = fmax(fmax(b2, o2), fmin(b1, o1));
            b1 = fmax(b1, o1);
        }
        double gs = p.group_top == 2 && per > 1 ? b1 + b2 : b1;
        if (gs != gs) gs = -INFINITY;
        int ahead = 0;                                       // groups that come before this lane's
        for (int g = 0; g < p.groups; g++) {
            const double other = __shfl_sync(0xffffffffu, gs, g * p.lanes);
            ahead += other > gs || (other == gs && g < group);
        }
        if (ahead >= p.top_groups) {
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
    for (int k = 0; k < p.top; k++) {
        const unsigned hi = (unsigned) (best >> 32), most = __reduce_max_sync(0xffffffffu, hi);
        const unsigned lo = hi == most ? (unsigned) best : 0u, most_lo = __reduce_max_sync(0xffffffffu, lo);
        const int e = hi == most && lo == most_lo ? first + at : 0x7fffffff;
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
    if (p.renorm) {
        double sum = lane < p.top ? mine : 0.0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += shfl_xor_f64(sum, o);
        mine = sum == 0.0 ? 0.0 : mine / sum;
    }
    if (lane < p.top) {
        p.ids[t * p.top + lane] = mine_e;
        p.wts[t * p.top + lane] = (float) (mine * p.scale);
    }
}

// Descending order of a lane's keys, by Batcher's odd-even merge sort.
template <int SLOTS> __device__ __forceinline__ void sort_keys(unsigned (&k)[SLOTS]) {
#pragma unroll
    for (int p = 1; p < SLOTS; p *= 2)
#pragma unroll
        for (int d = p; d >= 1; d /= 2)
#pragma unroll
            for (int j = d % p; j + d < SLOTS; j += 2 * d)
#pragma unroll
                for (int i = 0; i < d; i++)
                    if (i + j + d < SLOTS && (i + j) / (2 * p) == (i + j + d) / (2 * p)) {
                        const unsigned x = k[i + j], y = k[i + j + d];
                        k[i + j] = max(x, y);
                        k[i + j + d] = min(x, y);
                    }
}

// The same in 32 bits.  A sigmoid is off by less than 4e-7 (2 units in the last place each of the exponential and the reciprocal, which
// matter most at 1, and the rounding of the sum between them), a softmax by less than 5e-6 of the row's largest score (the exponentials'
// sum, 64 terms in a lane, has most of it), and the corrected score by half a unit of its own more.  Two of them whose order decides
// anything -- neighbours among the chosen and the first that is not, the last group taken and the first that is not -- may be nearer than twice
// that.  Outputs and groups are then put in order by their scores in 64 bits, an output or two a lane; more than one output at the border, softmax
// scores with a correction and scores that are no finite numbers leave the token to route_exact (whose latency, 5 us, was the whole call's as
// soon as one token in it took that way: 512 tokens 8.3 us, 61 tokens 2.9).
// Up to 8 outputs a lane, the lowest bits of a key give way to the output's slot (SLOTS units in the last place, which widen that border) and a
// lane sorts its keys: a choice is then a reduction and a step down the winner's list, a third of the instructions of looking at all of
// them again (8,192 tokens, 8 of 256: 17.5 us with that where sorted keys took 14.5); 16 and more outputs a lane are slower sorted (24 against 19).
template <int SLOTS>
__global__ void __launch_bounds__(128) moe_route_grouped_kernel(const RouteArgs p, int N, int vec) {
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const long long t = (long long) blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (t >= N) return;
    const int per = p.E / p.groups, group = lane / p.lanes, j0 = (lane - group * p.lanes) * p.chunk;
    const int first = group * per + j0, held = group < p.groups ? max(0, min(p.chunk, per - j0)) : 0;
    const float * z = p.logits + t * p.ld + first;
    float s[SLOTS], c[SLOTS];
#pragma unroll
    for (int i = 0; i < SLOTS; i++) { s[i] = -INFINITY; c[i] = 0.0f; }
    if (vec) {                                               // whole pieces of 16 bytes
#pragma unroll
        for (int i = 0; i + 3 < SLOTS; i += 4)
            if (i < held) {
                *reinterpret_cast<float4 *>(s + i) = *reinterpret_cast<const float4 *>(z + i);
                if (p.correction != nullptr) *reinterpret_cast<float4 *>(c + i) = __ldg(reinterpret_cast<const float4 *>(p.correction + first + i));
            }
    } else {
#pragma unroll
        for (int i = 0; i < SLOTS; i++)
            if (i < held) {
                s[i] = z[i];
                if (p.correction != nullptr) c[i] = __ldg(p.correction + first + i);
            }
    }
    float most = 0.0f;                                       // the row's largest score, or a bound of it
    float mx = -INFINITY;
    if (p.softmax) {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < SLOTS; i++) mx = fmaxf(mx, s[i]);
        mx = warp_max(mx);
#pragma unroll
        for (int i = 0; i < SLOTS; i++) {
            s[i] = __expf(s[i] - mx);
            sum += s[i];
        }
        most = __fdividef(1.0f, warp_sum(sum));
#pragma unroll
        for (int i = 0; i < SLOTS; i++) s[i] *= most;
    } else {
        most = 1.0f;
#pragma unroll
        for (int i = 0; i < SLOTS; i++) s[i] = route_sigmoid(s[i]);
    }
    constexpr bool SORT = SLOTS <= 8;
    constexpr unsigned SLOT_BITS = SORT ? SLOTS - 1 : 0;
    const float base = p.softmax ? 1e-5f : 2e-6f;
    auto number = [](unsigned k) { return __int_as_float((int) (k & 0x80000000u ? k ^ 0x80000000u : ~k)); };
    auto near_of = [&](float v) { return base * most + (base + (SORT ? SLOTS * 1.2e-7f : 0.0f)) * fabsf(v); };
    auto exact_score = [&](int e) {                          // of a sigmoid, or of a softmax without a correction as a multiple of the row's sum
        const double x = p.logits[t * p.ld + e];
        return p.softmax ? exp(x - (double) mx) : 1.0 / (1.0 + exp(-x)) + (p.correction != nullptr ? (double) p.correction[e] : 0.0);
    };
    unsigned key[SLOTS];                                     // 0: not to be chosen
#pragma unroll
    for (int i = 0; i < SLOTS; i++) key[i] = i < held ? (order_key(s[i] + c[i]) & ~SLOT_BITS) | (SLOT_BITS - (SORT ? i : 0)) : 0;
    unsigned k1 = 0, k2 = 0;                                 // this lane's two largest
    if constexpr (SORT) {
        sort_keys<SLOTS>(key);
        k1 = key[0];
        k2 = key[SLOTS > 1 ? 1 : 0];
    } else {
#pragma unroll
        for (int i = 0; i < SLOTS; i++) {
            k2 = max(k2, min(k1, key[i]));
            k1 = max(k1, key[i]);
        }
    }
    bool unsure = false;
    if (p.top_groups < p.groups) {
        for (int o = 1; o < p.lanes; o <<= 1) {
            const unsigned o1 = __shfl_xor_sync(0xffffffffu, k1, o), o2 = __shfl_xor_sync(0xffffffffu, k2, o);
            k2 = max(max(k2, o2), min(k1, o1));
            k1 = max(k1, o1);
        }
        const bool two = p.group_top == 2 && per > 1;
        const float gs = two ? number(k1) + number(k2) : number(k1);
        int ahead = 0;
        for (int g = 0; g < p.groups; g++) {
            const float other = __shfl_sync(0xffffffffu, gs, g * p.lanes);
            ahead += other > gs || (other == gs && g < group);
        }
        bool shut = ahead >= p.top_groups;
        const bool live = group < p.groups;
        const float lo = number(__reduce_min_sync(0xffffffffu, live && !shut ? order_key(gs) : 0xffffffffu));
        const float hi = number(__reduce_max_sync(0xffffffffu, live && shut ? order_key(gs) : 0u));
        // (the two that a group's score is made of may lie further from 0 than it does)
        const float widest = two ? fmaxf(fabsf(number(k1)), fabsf(number(k2))) : fabsf(gs);
        const bool border = live && !(lo - hi > 2.0f * near_of(widest));
        // (an infinity whose key holds a slot's number in its place is no number, which a maximum passes over: each by itself)
        unsure = live && !(fabsf(number(k1)) < 1e30f && (!two || fabsf(number(k2)) < 1e30f));
        if (__any_sync(0xffffffffu, border)) {
            // the groups again by the scores in 64 bits of each lane's two largest, where it is certain which these are
            if constexpr (SORT && SLOTS > 2) {
                const float third = number(key[2]), second = number(key[1]);
                unsure = unsure || (held > 2 && !(second - third > near_of(fmaxf(fabsf(second), fabsf(third))))) || (held > 0 && !(fabsf(number(key[0])) < 1e30f));
            }
            unsure = unsure || !SORT || (p.softmax && p.correction != nullptr);
            if (!__any_sync(0xffffffffu, unsure)) {
                double d1 = -INFINITY, d2 = -INFINITY;
#pragma unroll 1
                for (int i = 0; i < min(held, 2); i++) {
                    const double c64 = exact_score(first + (int) (SLOT_BITS - ((i == 0 ? key[0] : key[SLOTS > 1 ? 1 : 0]) & SLOT_BITS)));
                    d2 = fmax(d2, fmin(d1, c64));
                    d1 = fmax(d1, c64);
                }
                for (int o = 1; o < p.lanes; o <<= 1) {
                    const double o1 = shfl_xor_f64(d1, o), o2 = shfl_xor_f64(d2, o);
                    d2 = fmax(fmax(d2, o2), fmin(d1, o1));
                    d1 = fmax(d1, o1);
                }
                const double g64 = two ? d1 + d2 : d1;
                ahead = 0;
                for (int g = 0; g < p.groups; g++) {
                    const double other = __shfl_sync(0xffffffffu, g64, g * p.lanes);
                    ahead += other > g64 || (other == g64 && g < group);
                }
                shut = ahead >= p.top_groups;
            }
        }
        if (shut) {
#pragma unroll
            for (int i = 0; i < SLOTS; i++) key[i] = 0;
        }
    }
    // The chain: a lane holds its best key; the warp's best goes to choice k, and the lane that had it -- the first of them -- leaves its output's
    // number behind.  Two more than are taken: the first that is not, and how near the next one comes to it.
    __shared__ int taken[4][kGroupTopMost + 2];
    int * chosen = taken[threadIdx.x >> 5];
    unsigned best = key[0], mine_key = 0, edge_key = 0, beyond_key = 0;
    if constexpr (!SORT) {
#pragma unroll
        for (int i = 0; i < SLOTS; i++) best = max(best, key[i]);
    }
    for (int k = 0; k < p.top + 2; k++) {
        const unsigned won = __reduce_max_sync(0xffffffffu, best);
        if (lane == k) mine_key = won;
        if (k == p.top) edge_key = won;
        if (k == p.top + 1) beyond_key = won;
        if (won == 0) break;                                 // every output that there was is taken
        const unsigned who = __ballot_sync(0xffffffffu, best == won);
        if (lane == __ffs(who) - 1) {
            if constexpr (SORT) {
                chosen[k] = first + (int) (SLOT_BITS - (won & SLOT_BITS));
#pragma unroll
                for (int i = 0; i + 1 < SLOTS; i++) key[i] = key[i + 1];
                key[SLOTS - 1] = 0;
                best = key[0];
            } else {
                int at = 0;
                bool found = false;
                best = 0;
#pragma unroll
                for (int i = 0; i < SLOTS; i++) {
                    if (key[i] == won && !found) { key[i] = 0; at = i; found = true; }
                    best = max(best, key[i]);
                }
                chosen[k] = first + at;
            }
        }
    }
    __syncwarp();
    // which places are nearer to the one before than 32 bits can tell
    const float v = number(mine_key), before = __shfl_up_sync(0xffffffffu, v, 1);
    const bool there = lane <= p.top && mine_key != 0;
    const bool close = there && lane > 0 && v > -1e30f && !(before - v > near_of(fmaxf(fabsf(before), fabsf(v))));
    unsure = unsure || (lane < p.top && !(fabsf(v) < 1e30f));
    unsigned tied = __ballot_sync(0xffffffffu, close && lane < p.top);
    const float last = __shfl_sync(0xffffffffu, v, p.top - 1), edge = number(edge_key), beyond = number(beyond_key);
    if (edge_key != 0 && edge > -1e30f && !(last - edge > near_of(fmaxf(fabsf(last), fabsf(edge))))) {
        tied |= 1u;                                          // the first that is not may have to be; it cannot be told from more of them, nor has it
        unsure = unsure || p.top == 32 ||                    // a lane behind 32 choices
                 (beyond_key != 0 && beyond > -1e30f && !(edge - beyond > near_of(fmaxf(fabsf(edge), fabsf(beyond)))));
    }
    if (p.softmax && p.correction != nullptr && tied != 0) unsure = true;         // (would need the row's sum in 64 bits)
    unsure = __any_sync(0xffffffffu, unsure);
    int mine_e = there && !unsure ? chosen[lane] : 0;
    if (tied != 0 && !unsure) {
        // those that were chosen and the first that was not, put in the order that they have in 64 bits
        const double c64 = there ? exact_score(mine_e) : -INFINITY;
        int place = 0;
        for (int j = 0; j < min(p.top + 1, 32); j++) {
            const double other = __shfl_sync(0xffffffffu, c64, j);
            const int e = __shfl_sync(0xffffffffu, mine_e, j);
            place += other > c64 || (other == c64 && e < mine_e);
        }
        if (there) chosen[place] = mine_e;
        __syncwarp();
        mine_e = chosen[lane < p.top ? lane : 0];
    }
    // The chosen scores again, a lane each, for the weights: with the digits that the order could do without (an __expf is off by a unit in the
    // last place for every 0.85 of its argument), and a sigmoid in a form that does not overflow.  Scores of 32 bits end near e^-87: where a
    // smaller one has to be divided by the sum of the chosen, the token is done in 64.
    float mine = 0.0f;
    bool small = false;
    if (lane < p.top) {
        const float x = p.logits[t * p.ld + mine_e], d = p.softmax ? x - mx : x, e = expf(p.softmax ? d : -fabsf(x));
        mine = p.softmax ? e * most : (x < 0.0f ? e : 1.0f) / (1.0f + e);
        small = mine < 1e-36f && d > -750.0f;                // (below that 64 bits have nothing either)
    }
    if (p.renorm && __any_sync(0xffffffffu, small)) unsure = true;
    if (unsure) {
        route_exact<SLOTS>(p, t);
        return;
    }
    if (p.renorm) {
        const float sum = warp_sum(lane < p.top ? mine : 0.0f);
        mine = sum == 0.0f ? 0.0f : mine / sum;
    }
    if (lane < p.top) {
        p.ids[t * p.top + lane] = mine_e;
        p.wts[t * p.top + lane] = mine * (float) p.scale;
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
    RouteArgs p = {logits, ld, correction, E, groups, 32 / wide, 0, top_groups, group_top, top, softmax, renorm, (double) scale, ids, wts};
    const int per = E / groups, warps = 4;
    p.chunk = (per + p.lanes - 1) / p.lanes;
    const int vec = p.chunk % 4 == 0 && per % 4 == 0 && ld % 4 == 0 && (((uintptr_t) logits | (uintptr_t) correction) & 15) == 0;
    const dim3 grid((unsigned) (((long long) N + warps - 1) / warps));
    auto kernel = p.chunk <= 2 ? moe_route_grouped_kernel<2> : p.chunk <= 4 ? moe_route_grouped_kernel<4> : p.chunk <= 8 ? moe_route_grouped_kernel<8>
                : p.chunk <= 16 ? moe_route_grouped_kernel<16> : p.chunk <= 32 ? moe_route_grouped_kernel<32>
                : moe_route_grouped_kernel<64>;              // 17 groups of 60: half of the lanes hold nothing
    return iian_launch(kernel, grid, dim3(warps * 32), 0, stream, p, N, vec);
}
