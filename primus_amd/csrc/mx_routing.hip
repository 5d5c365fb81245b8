// Routing of tokens to experts and its gradient: what stands in front of the expert MLP
// (primus/backends/megatron/core/transformer/experts.py:24-268 takes rows that a router has assigned).
//
// Per token, from its logits l[E]:
//   s = softmax(l) or sigmoid(l),  c = s + expert_bias  (the bias takes part in the choice only)
//   with groups: an expert group's score is the sum of its topk / group_topk largest c; the group_topk best groups stay
//   indices = the topk largest c, best first, ties to the lower index
//   probs   = scale * s[indices], renormalised over the chosen ones if asked
// and over all tokens the number of tokens of every expert.
//
// Bound by instructions and, for few tokens, by one row's chain of them: a row is held in registers by LPR lanes of a wave, V logits a
// lane, sorted inside the lane once (V = 4: five comparisons), and a round of the choice is one maximum over the row's lanes and a step
// in one lane's list, 27 instructions.  Without bias and groups the order of the scores is that of the logits, which are compared as they are.
// With them the scores are compared in fp32 first; a row in which two neighbours of the result, or the last chosen and the best
// left out that is no true tie of it (same logit, same bias), are nearer to each other than the rounding of fp32 scores allows to tell apart is
// chosen again from scores in fp64 (one row in 2000 at 256 fp32 scores), so the indices are those of the definition and not of a rounding.
// A tie at that border costs its row a pass over the registers: 16384 rows of 256 zeros 21.0 us with the counts, 19.2 without the comparison.
//
// us in a trace: 8 tokens of 128 experts, top 4, 2.9; 16384 of 8, top 2, 3.6 and 2.3 for adding up the counts, gradient 3.6; 5003 of 160, top 6,
// 9.4 + 3.3, 7.2; 16384 of 256, sigmoid, bias, 4 of 8 groups, top 8, 29 + 3.9, 7.0 (the logits alone are 3.3 at the rate of a large copy).  The last one's forward
// without the fp64 rows is 22-26, with one round instead of nine 17.
#include "mx_lanes.h"

namespace mxl {

constexpr int RT_MAX_EXPERTS = MXL_MAX_GROUPS;
constexpr int RT_MAX_TOPK = 32;
constexpr int RT_MAX_EXPERT_GROUPS = 64;

struct RouteArgs {
    const void* logits;
    const float* bias;          // null: none
    const uint8_t* mask;        // null: every token is routed
    float* probs;
    int64_t* indices;
    int64_t* counts;            // written by the launch itself where it is one workgroup, else
    int* partial;               // [workgroups, experts], summed by a second launch
    int64_t tokens;
    int experts, topk, dtype, sigmoid, renorm;
    int groups, group_topk, group_size, lanes_per_group, take;
    float scale;
};

// Unsigned key in the order of the float: NaN 1 (below -inf), 0 is left for "no element here"; -0 and 0 are the same.
__device__ __forceinline__ uint32_t order_key(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);
    const uint32_t k = (b >> 31) ? ~b : b | 0x80000000u;
    return x != x ? 1u : k;
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float((k >> 31) ? k & 0x7FFFFFFFu : ~k); }

// A softmax over nothing but -inf (every expert of the row disabled, or every chosen one) is 0 everywhere.
__device__ __forceinline__ float finite_top(float top) { return top == -INFINITY ? 0.f : top; }
__device__ __forceinline__ float some(float sum) { return sum == 0.f ? 1.f : sum; }
__device__ __forceinline__ float sigmoid_of(float x) { return 1.f / (1.f + expf(-x)); }
// the same for the choice: hardware exp2 and reciprocal, about 1 ulp each; the product with log2 e adds 1.45 |x| 2^-24
__device__ __forceinline__ float exp_fast(float x) { return __builtin_amdgcn_exp2f(x * 1.4426950408889634f); }
__device__ __forceinline__ float sigmoid_fast(float x) { return __builtin_amdgcn_rcpf(1.f + exp_fast(-x)); }
__device__ __forceinline__ uint32_t dpp_next_lane(uint32_t v) {        // lane l: lane l + 1's; the last lane 0
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x130, 0xF, 0xF, true);      // wave_shl 1
}
__device__ __forceinline__ float dpp_next_lane(float v) { return __uint_as_float(dpp_next_lane(__float_as_uint(v))); }
// Largest of the wave's 64 keys as a scalar: inside the rows of 16 lanes, then row 0 into 1 and 2 into 3, 1 into 3; lane 63 has it.
// (Six instructions; with every lane given the result the last two steps are four each.)
__device__ __forceinline__ uint32_t wave_max_key(uint32_t v) {
    v = lanes_reduce<OpMaxU, 16>(v);
    v = OpMaxU::f(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xA, 0xF, false));      // row_bcast 15
    v = OpMaxU::f(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xC, 0xF, false));      // row_bcast 31
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// (key, expert) pairs of a lane in descending order, equal keys by ascending index: Batcher's odd-even merge sort
template <int V> __device__ __forceinline__ void sort_pairs(uint32_t (&key)[V], uint32_t (&idx)[V]) {
    auto order = [&](int a, int b) __attribute__((always_inline)) {      // a < b: the better one to a
        const bool keep = key[a] > key[b] || (key[a] == key[b] && idx[a] < idx[b]);
        const uint32_t ka = key[a], ia = idx[a];
        key[a] = keep ? ka : key[b];
        idx[a] = keep ? ia : idx[b];
        key[b] = keep ? key[b] : ka;
        idx[b] = keep ? idx[b] : ia;
    };
#pragma unroll
    for (int p = 1; p < V; p <<= 1)
#pragma unroll
        for (int k = p; k >= 1; k >>= 1)
#pragma unroll
            for (int j = k % p; j + k < V; j += 2 * k)
#pragma unroll
                for (int i = 0; i < k; ++i)
                    if (i + j + k < V && (i + j) / (2 * p) == (i + j + k) / (2 * p)) order(i + j, i + j + k);
}
template <int V> __device__ __forceinline__ void pop_head(uint32_t (&key)[V], uint32_t (&idx)[V], bool take) {
#pragma unroll
    for (int v = 0; v + 1 < V; ++v) {
        key[v] = take ? key[v + 1] : key[v];
        idx[v] = take ? idx[v + 1] : idx[v];
    }
    key[V - 1] = take ? 0u : key[V - 1];
}

// The choice of one row again, by a whole wave, from scores in fp64, given the lane's logits (-inf past `have`) and the row's largest;
// lane k < topk returns the k-th index.  Rare, but the wave that does it is the one the launch waits for: the scores' order keys stand
// in the wave's LDS, a lane keeps its best one in registers, and a round is two scalar maxima (upper, then lower halves).
template <int V>
__device__ __forceinline__ int choose_fp64(const RouteArgs& p, const float (&l)[V], const float* bias, float top, int first, int have, uint64_t* keys) {
    const int lane = threadIdx.x & 63;
    double sum = 0.0;
    if (!p.sigmoid) {
        _Pragma("unroll 1") for (int v = 0; v < V; ++v) sum += v < have ? exp((double)l[v] - (double)top) : 0.0;
        for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
        sum = sum == 0.0 ? 1.0 : sum;
    }
    _Pragma("unroll 1") for (int v = 0; v < V; ++v) {
        double x = (double)l[v];
        x = (p.sigmoid ? 1.0 / (1.0 + exp(-x)) : exp(x - (double)top) / sum) + (double)bias[v < have ? first + v : 0];
        const uint64_t bits = (uint64_t)__double_as_longlong(x + 0.0);
        const uint64_t k = (bits >> 63) ? ~bits : bits | ((uint64_t)1 << 63);
        keys[v * 64 + lane] = v >= have ? 0 : x != x ? 1 : k;       // 0: no element, 1: NaN, below -inf
    }
    uint32_t left = have >= 32 ? 0xFFFFFFFFu : (1u << have) - 1u;   // this lane's elements that are still to be had
    uint64_t best = 0;
    int at = 0;
    auto rescan = [&](uint32_t have_bits) {
        best = 0;
        _Pragma("unroll 1") for (int v = 0; v < V; ++v) {
            const uint64_t k = keys[v * 64 + lane];
            if (((have_bits >> v) & 1) && k > best) best = k, at = v;
        }
    };
    rescan(left);
    if (p.groups > 1) {
        uint32_t have_bits = left;
        double score = 0.0;
        for (int i = 0; i < p.take; ++i) {
            const uint32_t hi = lanes_reduce<OpMaxU>((uint32_t)(best >> 32), p.lanes_per_group);
            const uint32_t lo = lanes_reduce<OpMaxU>((uint32_t)(best >> 32) == hi ? (uint32_t)best : 0u, p.lanes_per_group);
            const uint64_t k = (uint64_t)hi << 32 | lo;
            const uint32_t who = lanes_reduce<OpMinU>(best == k ? (uint32_t)lane : 64u, p.lanes_per_group);
            if (k != 0) score += __longlong_as_double((long long)((k >> 63) ? k & ~((uint64_t)1 << 63) : ~k));
            if (who == (uint32_t)lane && k != 0) {
                have_bits &= ~(1u << at);
                rescan(have_bits);
            }
        }
        const bool nan = score != score;        // behind every score that is none
        int ahead = 0;
        const int grp = lane / p.lanes_per_group;
        for (int g = 0; g < p.groups; ++g) {
            const double other = __shfl(score, g * p.lanes_per_group);
            ahead += other > score || (nan ? g < grp || other == other : other == score && g < grp);
        }
        if (ahead >= p.group_topk) left = 0;
        rescan(left);
    }
    int mine = 0;
    for (int k = 0; k < p.topk; ++k) {
        const uint32_t hi = wave_max_key((uint32_t)(best >> 32));
        const uint32_t lo = wave_max_key((uint32_t)(best >> 32) == hi ? (uint32_t)best : 0u);
        const int who = __builtin_ctzll(__ballot(best == ((uint64_t)hi << 32 | lo)));      // the lower index is in the lower lane
        const int won = __builtin_amdgcn_readlane(first + at, who);
        mine = lane == k ? won : mine;
        if (lane == who) {
            left &= ~(1u << at);
            rescan(left);
        }
    }
    return mine;
}

// SCORED: bias or groups, so scores are computed and compared (a row per wave); otherwise the logits are.
template <int V, bool SCORED> constexpr int route_waves() { return !SCORED ? 16 : V <= 8 ? 8 : 64 / V; }

template <int LPR, int V, bool SCORED>
__global__ __launch_bounds__((route_waves<V, SCORED>() * 64), (V > 4 ? 1 : SCORED ? 6 : 8)) void route_fwd_kernel(RouteArgs p) {
    static_assert(!SCORED || LPR == 64, "a scored row is a wave's");
    constexpr int WAVES = route_waves<V, SCORED>(), RPW = 64 / LPR;
    __shared__ int hist[RT_MAX_EXPERTS];
    __shared__ float bias[SCORED ? RT_MAX_EXPERTS : 1];
    __shared__ uint64_t spare[SCORED ? WAVES * V * 64 : 1];
    const int t = threadIdx.x, w = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63, lr = lane & (LPR - 1);
    for (int e = t; e < p.experts; e += WAVES * 64) {
        hist[e] = 0;
        if (SCORED) bias[e] = p.bias ? p.bias[e] : 0.f;
    }
    __syncthreads();
    // element (lane, v) of a row: expert `first + v`, if v < have.  Lower experts sit in lower lanes.
    int first, have;
    if (SCORED) {
        const int sub = lr & (p.lanes_per_group - 1), g = lr / p.lanes_per_group;
        first = g * p.group_size + sub * V;
        have = g < p.groups ? p.group_size - sub * V : 0;
    } else {
        first = lr * V;
        have = p.experts - first;
    }
    have = have < 0 ? 0 : have > V ? V : have;

    const int64_t step = (int64_t)gridDim.x * WAVES * RPW;
    auto fetch = [&](int64_t row0, float (&l)[V]) __attribute__((always_inline)) {
        const int64_t row = LPR == 64 ? row0 : row0 + lane / LPR, base = (row < p.tokens ? row : p.tokens - 1) * p.experts;
#pragma unroll
        for (int v = 0; v < V; ++v) l[v] = v < have ? load_dt(p.logits, p.dtype, base + first + v) : -INFINITY;
    };
    int64_t row0 = ((int64_t)blockIdx.x * WAVES + w) * RPW;
    float next[V];
    if (row0 < p.tokens) fetch(row0, next);
    for (; row0 < p.tokens; row0 += step) {
        const int64_t row = LPR == 64 ? row0 : row0 + lane / LPR;
        const bool in = row < p.tokens;
        float l[V];
#pragma unroll
        for (int v = 0; v < V; ++v) l[v] = next[v];
        if (row0 + step < p.tokens) fetch(row0 + step, next);       // the next row's logits travel while this one's are looked at
        const bool routed = !p.mask || !in || p.mask[row];

        float top = 0.f, total = 1.f;           // of the row: largest logit, sum of exp(l - top)
        if (!p.sigmoid && (SCORED || !p.renorm)) {
            top = -INFINITY;
#pragma unroll
            for (int v = 0; v < V; ++v) top = fmaxf(top, l[v]);
            top = finite_top(lanes_max<LPR>(top));
            float s = 0.f;
#pragma unroll
            for (int v = 0; v < V; ++v) s += v < have ? exp_fast(l[v] - top) : 0.f;
            total = some(lanes_sum<LPR>(s));
        }
        // What two fp32 scores may be off together: sigmoid, at most 2^-22 each (an exponential, a sum, a reciprocal).  Softmax: a
        // score s = exp(-x) / total is off by s (1.45 x + 60) 2^-24 (the exponentials, V + 6 additions, the quotient), and neither s
        // nor 2 s x passes 1 / total.  Without a bias nothing left out has a larger score than what it is compared with: relative there.
        const float pair_off = p.sigmoid ? 0x1p-21f : 0x1p-17f / total;
        uint32_t key[V], idx[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float x = l[v];
            if (SCORED && v < have) x = (p.sigmoid ? sigmoid_fast(l[v]) : exp_fast(l[v] - top) / total) + bias[first + v];
            key[v] = v < have ? order_key(x) : 0u;
            idx[v] = (uint32_t)(first + v);
        }
        sort_pairs<V>(key, idx);
        bool doubt = false, keep = true;
        if (SCORED && p.groups > 1) {
            uint32_t gk[V], gi[V];
#pragma unroll
            for (int v = 0; v < V; ++v) gk[v] = key[v], gi[v] = 0u;
            float score = 0.f, terms = 0.f;         // the group's sum, and its terms' magnitudes
            for (int i = 0; i < p.take; ++i) {
                const uint32_t best = lanes_reduce<OpMaxU>(gk[0], p.lanes_per_group);
                const uint32_t who = lanes_reduce<OpMinU>(gk[0] == best ? (uint32_t)lane : 64u, p.lanes_per_group);
                score += best ? key_value(best) : 0.f;
                terms += best ? fabsf(key_value(best)) : 0.f;
                pop_head<V>(gk, gi, who == (uint32_t)lane && best != 0u);
            }
            int ahead = 0;
            for (int g = 0; g < p.groups; ++g)
                ahead += __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(score), g * p.lanes_per_group)) > score;
            keep = ahead < p.group_topk;
            const bool real = lane / p.lanes_per_group < p.groups;
            if (p.group_topk < p.groups) {
                // The worst that any group kept may be and the best that any left out may be; groups of the same score and groups that are
                // NaN, of which too many are kept, are told apart in fp64.  A sum of n = take terms is off by what its scores are, and by n roundings at most
                // where biases are added and as many in the sum, each up to 2^-24 of the terms' magnitudes together (biased terms may
                // cancel: the sum says nothing of them).  Of a softmax without a bias terms below 2^-126 may be 0, at most 32 of them.  Infinite
                // sums are exact.
                const float sum_off = (p.bias || p.sigmoid ? 0.5f * pair_off * (float)p.take : fmaf(0x1p-16f, score, 0x1p-121f)) + 0x1p-22f * (float)p.take * terms;
                const float off = fabsf(score) == INFINITY ? 0.f : sum_off;
                const int kept = __builtin_popcountll(__ballot(keep && real)) / p.lanes_per_group;
                const float in_worst = key_value(~wave_max_key(real && keep ? ~order_key(score - off) : 0u));
                const float out_best = key_value(wave_max_key(real && !keep ? order_key(score + off) : 0u));
                doubt = kept != p.group_topk || !(in_worst > out_best);
            }
#pragma unroll
            for (int v = 0; v < V; ++v) key[v] = keep ? key[v] : 0u;
        }
        // the choice, one expert a round; lane k of the row keeps the k-th (a scored row looks one further, to compare with it)
        int mine = 0;
        uint32_t mine_key = 0u;
        const int rounds = p.topk + (SCORED ? 1 : 0);
        for (int k = 0; k < rounds; ++k) {
            if constexpr (LPR == 64) {
                const uint32_t best = wave_max_key(key[0]);
                const uint64_t hit = __ballot(key[0] == best), low = hit & (0 - hit);       // equal keys: the lower index is in the lower lane
                const int won = __builtin_amdgcn_readlane((int)idx[0], __builtin_ctzll(hit));
                const bool kth = __builtin_amdgcn_inverse_ballot_w64((uint64_t)1 << k);
                mine = kth ? won : mine;
                mine_key = kth ? best : mine_key;
                pop_head<V>(key, idx, __builtin_amdgcn_inverse_ballot_w64(low));
            } else {
                const uint32_t best = lanes_reduce<OpMaxU, LPR>(key[0]);
                const uint32_t won = lanes_reduce<OpMinU, LPR>(key[0] == best ? idx[0] : 0xFFFFFFFFu);
                mine = lr == k ? (int)won : mine;
                mine_key = lr == k ? best : mine_key;
                pop_head<V>(key, idx, key[0] == best && idx[0] == won);
            }
        }
        // lane k < topk: its expert's logit (an unscored row's is its key's value: exact, but for a NaN, which stays one)
        const bool chosen = lr < p.topk;
        float ml;
        if constexpr (SCORED) {
            const int64_t at = (in ? row : p.tokens - 1) * p.experts;
            ml = mine_key ? load_dt(p.logits, p.dtype, at + mine) : -INFINITY;
            const float b = bias[mine_key ? mine : 0], s = p.sigmoid ? sigmoid_fast(ml) : exp_fast(ml - top) / total, c = key_value(mine_key);
            const float nl = dpp_next_lane(ml), ns = dpp_next_lane(s), nc = dpp_next_lane(c), nb = dpp_next_lane(b);
            const uint32_t nk = dpp_next_lane(mine_key);
            auto off_of = [&](float both, float c1, float c2) __attribute__((always_inline)) {
                return (p.bias || p.sigmoid ? pair_off : 0x1p-16f * both) + 0x1p-23f * (fabsf(c1) + fabsf(c2));
            };
            // nothing follows, or the same logit and bias (a true tie), or far enough apart: told rightly
            const bool tie = nk != 0u && ml == nl && b == nb;
            const bool told = !chosen || nk == 0u || tie || c - nc > off_of(s + ns, c, nc);
            // The last one chosen and the first left out are a true tie: the best one left out that is none of their kind has to be told from
            // them too.  True ties have the same fp32 key; whether anything else has it, the numbers of both say.
            if (__ballot(tie) >> (p.topk - 1) & 1) {
                auto of_last = [&](float x) { return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(x), p.topk - 1)); };
                const uint32_t key_t = (uint32_t)__builtin_amdgcn_readlane((int)mine_key, p.topk - 1);
                const float l_t = of_last(ml), b_t = of_last(b), c_t = of_last(c);
                uint32_t behind = 0u;
                int others = mine_key == key_t;         // chosen or left out, with that key, less the ties
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    behind = key[v] < key_t && key[v] > behind ? key[v] : behind;
                    others += (key[v] == key_t) - (v < have && keep && l[v] == l_t && bias[first + v] == b_t);
                }
                behind = wave_max_key(behind);
                const float z = key_value(behind);      // (the score itself where there is no bias)
                doubt |= lanes_sum<64>((float)others) != 0.f || (behind != 0u && !(c_t - z > off_of(c_t + z, c_t, z)));
            }
            doubt = __any(doubt || !told);
            if (doubt) {
                mine = choose_fp64<V>(p, l, bias, top, first, have, spare + w * V * 64);
                ml = chosen ? load_dt(p.logits, p.dtype, at + mine) : -INFINITY;
            }
            ml = chosen ? ml : -INFINITY;
        } else {
            ml = chosen ? key_value(mine_key) : -INFINITY;
        }
        float prob;
        if (p.sigmoid) {
            const float s = chosen ? sigmoid_of(ml) : 0.f;
            prob = p.renorm ? s / (lanes_sum<LPR>(s) + 1e-20f) : s;
        } else if (p.renorm) {
            const float m = finite_top(lanes_max<LPR>(ml));
            const float s = chosen ? expf(ml - m) : 0.f;
            prob = s / some(lanes_sum<LPR>(s));
        } else {
            prob = expf(ml - top) / total;
        }
        if (in && chosen) {
            p.probs[row * p.topk + lr] = routed ? prob * p.scale : 0.f;
            p.indices[row * p.topk + lr] = routed ? mine : -1;
            if (routed) atomicAdd(&hist[mine], 1);
        }
    }
    __syncthreads();
    if (gridDim.x == 1) {
        for (int e = t; e < p.experts; e += WAVES * 64) p.counts[e] = hist[e];
    } else {
        for (int e = t; e < p.experts; e += WAVES * 64) p.partial[(int64_t)blockIdx.x * p.experts + e] = hist[e];
    }
}

// counts[e] = sum over the workgroups: 16 experts by 64 runs of workgroups, 8 loads on their way
__global__ __launch_bounds__(1024) void route_counts_kernel(const int* partial, int blocks, int experts, int64_t* counts) {
    __shared__ int part[64][17];
    const int lane = threadIdx.x & 15, run = threadIdx.x >> 4, e = blockIdx.x * 16 + lane;
    int n = 0;
    if (e < experts) {
        for (int b0 = run; b0 < blocks; b0 += 64 * 8) {
            int x[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) x[u] = b0 + 64 * u < blocks ? partial[(int64_t)(b0 + 64 * u) * experts + e] : 0;
#pragma unroll
            for (int u = 0; u < 8; ++u) n += x[u];
        }
    }
    part[run][lane] = n;
    __syncthreads();
    if (run == 0 && e < experts) {
        int64_t total = 0;
#pragma unroll
        for (int i = 0; i < 64; ++i) total += part[i][lane];
        counts[e] = total;
    }
}

struct RouteBwdArgs {
    const float* dprobs;
    const void* logits;
    const int64_t* indices;
    void* dlogits;
    int64_t tokens;
    int experts, topk, dtype, sigmoid, renorm;
    float scale;
};

// g = scale * dprobs, w = the chosen scores' shares.  Renormalised: dl = w (g - sum w g) at the chosen experts (softmax),
// (g - sum w g) / (S + 1e-20) * s (1 - s) (sigmoid); as they are: softmax s_e ([e chosen] g_e - sum s g) at every expert,
// sigmoid g s (1 - s).  The chosen experts' gradients meet their rows through LDS, which is zero between rows.
constexpr int RB_WAVES = 8;
// All but the plain softmax: the other experts' gradients are zero.  LPR lanes a row, so that 64 / LPR rows wait for their indices and
// logits together; the rows leave as one run of memory, four elements a lane and request (VEC).  Bound by that one wait and, with many
// experts, by the rows' bytes.  us from launch to launch of a replayed graph (a trace has 0.5 to 1 us more for a launch) with a wave a row, two
// rows, eight rows: 16384 tokens of 8 experts, top 2, 5.8 / 4.4 / 2.9, of 64, top 6, 6.2 / 4.8 / 3.8, of 256, top 8, 8.7 / 6.1 / 6.5, of
// 1024 16.2 / 13.6 / 16.2; 8192 of 64 4.5 / 3.6 / 3.4; 1024 of 64 2.8 / 2.8 / 3.2, of 256 3.3 / 3.1 / 4.0.  So eight rows for many tokens of few
// experts, else two.
template <int LPR, bool VEC>
__global__ __launch_bounds__(RB_WAVES * 64) void route_bwd_chosen_kernel(RouteBwdArgs p) {
    constexpr int RPW = 64 / LPR;
    extern __shared__ __attribute__((aligned(16))) float lds[];
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, lr = lane & (LPR - 1), sub = lane / LPR;
    const int size = RPW * p.experts;
    float* d = lds + w * ((size + 3) & ~3);
    for (int e = lane * 4; e < size; e += 256) *(v4f*)(d + e) = v4f{0.f, 0.f, 0.f, 0.f};      // (a wave's part is a multiple of four long)
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    for (int64_t row0 = ((int64_t)blockIdx.x * RB_WAVES + w) * RPW; row0 < p.tokens; row0 += (int64_t)gridDim.x * RB_WAVES * RPW) {
        const int64_t row = row0 + sub;
        const int64_t at = row < p.tokens && lr < p.topk ? p.indices[row * p.topk + lr] : -1;
        const bool chosen = at >= 0 && at < p.experts;
        const float g = chosen ? p.dprobs[row * p.topk + lr] * p.scale : 0.f;
        const float ml = chosen ? load_dt(p.logits, p.dtype, row * p.experts + at) : -INFINITY;
        float mine;
        if (p.sigmoid) {
            const float s = chosen ? sigmoid_of(ml) : 0.f;
            float ds = g;
            if (p.renorm) {
                const float sum = lanes_sum<LPR>(s) + 1e-20f;
                ds = (g - lanes_sum<LPR>(g * (s / sum))) / sum;
            }
            mine = ds * s * (chosen ? sigmoid_of(-ml) : 0.f);      // 1 - s without cancellation
        } else {
            const float m = finite_top(lanes_max<LPR>(ml));
            const float e = chosen ? expf(ml - m) : 0.f;
            const float wgt = e / some(lanes_sum<LPR>(e));
            mine = wgt * (g - lanes_sum<LPR>(wgt * g));
        }
        float* mine_at = d + sub * p.experts + (chosen ? (int)at : 0);
        if (chosen) atomicAdd(mine_at, mine);      // the same expert twice in a row: its gradients add up
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        const int n = (int)((p.tokens - row0 < RPW ? p.tokens - row0 : RPW) * p.experts), whole = VEC ? n & ~3 : 0;
        const int64_t base = row0 * p.experts;
        if constexpr (VEC) {
            for (int e = lane * 4; e < whole; e += 256) {
                const v4f x = *(const v4f*)(d + e);
                if (p.dtype == MXL_DT_F32) {
                    *(v4f*)((float*)p.dlogits + base + e) = x;
                } else {
                    typedef _Float16 h4 __attribute__((ext_vector_type(4)));
                    const h4 h = {(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3]};
                    const uint2 b = make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]));
                    *(uint2*)((uint16_t*)p.dlogits + base + e) = p.dtype == MXL_DT_BF16 ? b : __builtin_bit_cast(uint2, h);
                }
            }
        }
        for (int e = whole + lane; e < n; e += 64) store_dt(p.dlogits, p.dtype, base + e, d[e]);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (chosen) *mine_at = 0.f;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

// The plain softmax: a wave a row, whose logits are read again
__global__ __launch_bounds__(RB_WAVES * 64) void route_bwd_kernel(RouteBwdArgs p) {
    __shared__ float rows[RB_WAVES][RT_MAX_EXPERTS];
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
    float* d = rows[w];
    for (int e = lane; e < p.experts; e += 64) d[e] = 0.f;
    for (int64_t row = (int64_t)blockIdx.x * RB_WAVES + w; row < p.tokens; row += (int64_t)gridDim.x * RB_WAVES) {
        const int64_t base = row * p.experts;
        const int64_t at = lane < p.topk ? p.indices[row * p.topk + lane] : -1;
        const bool chosen = at >= 0 && at < p.experts;
        const float ml = chosen ? load_dt(p.logits, p.dtype, base + at) : -INFINITY;
        const float g = chosen ? p.dprobs[row * p.topk + lane] * p.scale : 0.f;
        float top = -INFINITY, sum = 0.f;
        for (int e = lane; e < p.experts; e += 64) top = fmaxf(top, load_dt(p.logits, p.dtype, base + e));
        top = finite_top(lanes_max<64>(top));
        for (int e = lane; e < p.experts; e += 64) sum += expf(load_dt(p.logits, p.dtype, base + e) - top);
        const float total = some(lanes_sum<64>(sum));
        const float s = chosen ? expf(ml - top) / total : 0.f, all = lanes_sum<64>(s * g);
        const bool live = __any(chosen);
        if (chosen) atomicAdd(&d[at], s * g);      // the same expert twice in a row: its gradients add up
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        for (int e = lane; e < p.experts; e += 64) {
            float x = d[e];
            if (live) x -= expf(load_dt(p.logits, p.dtype, base + e) - top) / total * all;
            store_dt(p.dlogits, p.dtype, base + e, x);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (chosen) d[at] = 0.f;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

template <int LPR> static void launch_route_bwd_chosen(const RouteBwdArgs& a, hipStream_t st) {
    constexpr int RPW = 64 / LPR;
    const int lds = RB_WAVES * ((RPW * a.experts + 3) & ~3) * 4;       // at most 64 KiB: two rows of 1024, or eight of 64, a wave
    int64_t blocks = (a.tokens + RB_WAVES * RPW - 1) / (RB_WAVES * RPW);
    if (blocks > 4096) blocks = 4096;
    // a wave's rows start at a multiple of four elements
    const bool vec = RPW * a.experts % 4 == 0 && ((uintptr_t)a.dlogits & (a.dtype == MXL_DT_F32 ? 15 : 7)) == 0;
    const dim3 grid((unsigned)blocks), block(RB_WAVES * 64);
    if (vec) hipLaunchKernelGGL((route_bwd_chosen_kernel<LPR, true>), grid, block, (unsigned)lds, st, a);
    else hipLaunchKernelGGL((route_bwd_chosen_kernel<LPR, false>), grid, block, (unsigned)lds, st, a);
}

// workgroups of a forward launch: rows for every wave slot of the chip at most; a few tokens are one, which writes the counts itself.  Where
// a wave takes several rows that is up to two rounds of rows, on the GPU / host, against two launches: 64 tokens of 128 experts 6.8 / 12.2
// and 6.8 / 14.7 us, 256 of 8 3.5 / 12.3 and 4.6 / 14.8; a third and fourth round cost more than the launch (128 of 128 11.7 and 6.9), and so does a
// second one of rows that are a wave's (32 of 256 9.2 and 8.0).
static int64_t route_blocks(int64_t tokens, int rows_per_block, int rows_per_wave = 1) {
    if (tokens <= 16 || (rows_per_wave > 1 && tokens <= 2 * rows_per_block)) return 1;
    int64_t b = (tokens + rows_per_block - 1) / rows_per_block;
    return b < 768 ? b : 768;
}

template <int LPR, int V, bool SCORED>
static int launch_route(const RouteArgs& a, hipStream_t st) {
    constexpr int WAVES = route_waves<V, SCORED>();
    const int64_t blocks = route_blocks(a.tokens, WAVES * (64 / LPR), 64 / LPR);
    hipLaunchKernelGGL((route_fwd_kernel<LPR, V, SCORED>), dim3((unsigned)blocks), dim3(WAVES * 64), 0, st, a);
    if (blocks > 1)
        hipLaunchKernelGGL(route_counts_kernel, dim3((unsigned)((a.experts + 15) / 16)), dim3(1024), 0, st, a.partial, (int)blocks, a.experts, a.counts);
    return hipGetLastError() == hipSuccess ? MXL_OK : MXL_ELAUNCH;
}

static bool route_sizes_ok(int64_t tokens, int experts, int topk, int dtype, int score) {
    return tokens >= 0 && tokens <= 0x7FFFFFFF && experts >= 1 && experts <= RT_MAX_EXPERTS && topk >= 1 && topk <= RT_MAX_TOPK && topk <= experts &&
           dtype >= MXL_DT_F32 && dtype <= MXL_DT_F16 && (score == MXL_SCORE_SOFTMAX || score == MXL_SCORE_SIGMOID);
}

__global__ void route_zero_counts_kernel(int64_t* counts, int experts) {
    for (int e = threadIdx.x; e < experts; e += 256) counts[e] = 0;
}

}  // namespace mxl

using namespace mxl;

extern "C" int64_t mxl_topk_routing_workspace_bytes(int64_t tokens, int experts) {
    if (tokens < 0 || experts < 1 || experts > RT_MAX_EXPERTS) return -1;
    const int64_t blocks = route_blocks(tokens, 2);        // (two rows at least in any of the kernels)
    return blocks > 1 ? blocks * experts * 4 : 0;
}

extern "C" int mxl_topk_routing(const void* logits, int dtype, int64_t tokens, int experts, int topk, int score, const float* expert_bias,
                                int num_groups, int group_topk, int renormalize, float scale, const uint8_t* token_mask, float* probs,
                                int64_t* indices, int64_t* counts, void* workspace, int64_t workspace_bytes, void* stream) {
    if (!route_sizes_ok(tokens, experts, topk, dtype, score) || !counts) return MXL_EINVAL;
    if (num_groups < 1 || num_groups > RT_MAX_EXPERT_GROUPS || experts % num_groups != 0 || group_topk < 1 || group_topk > num_groups ||
        topk > group_topk * (experts / num_groups))
        return MXL_EINVAL;
    if (tokens > 0 && (!logits || !probs || !indices)) return MXL_EINVAL;
    const int64_t need = mxl_topk_routing_workspace_bytes(tokens, experts);
    if (need > 0 && (workspace_bytes < need || !workspace)) return MXL_EINVAL;
    if (!device_is_gfx950()) return MXL_ENODEV;
    hipStream_t st = (hipStream_t)stream;
    if (tokens == 0) {
        hipLaunchKernelGGL(route_zero_counts_kernel, dim3(1), dim3(256), 0, st, counts, experts);
        return hipGetLastError() == hipSuccess ? MXL_OK : MXL_ELAUNCH;
    }
    RouteArgs a{};
    a.logits = logits, a.bias = expert_bias, a.mask = token_mask, a.probs = probs, a.indices = indices, a.counts = counts;
    a.partial = (int*)workspace, a.tokens = tokens, a.experts = experts, a.topk = topk, a.dtype = dtype;
    a.sigmoid = score == MXL_SCORE_SIGMOID, a.renorm = renormalize != 0, a.scale = scale;
    a.groups = num_groups, a.group_topk = group_topk, a.group_size = experts / num_groups;
    // the topk / group_topk best of a group make its score
    a.take = topk / group_topk < 1 ? 1 : topk / group_topk;
    if (a.take > a.group_size) a.take = a.group_size;
    if (expert_bias || num_groups > 1) {
        int pow2 = 1;
        while (pow2 < num_groups) pow2 *= 2;
        a.lanes_per_group = 64 / pow2;
        const int v = (a.group_size + a.lanes_per_group - 1) / a.lanes_per_group;
        if (v <= 1) return launch_route<64, 1, true>(a, st);
        if (v <= 2) return launch_route<64, 2, true>(a, st);
        if (v <= 4) return launch_route<64, 4, true>(a, st);
        if (v <= 8) return launch_route<64, 8, true>(a, st);
        if (v <= 16) return launch_route<64, 16, true>(a, st);
        return launch_route<64, 32, true>(a, st);
    }
    a.lanes_per_group = 64;
    if (topk <= 8 && experts <= 8) return launch_route<8, 1, false>(a, st);
    if (topk <= 8 && experts <= 16) return launch_route<8, 2, false>(a, st);
    if (topk <= 8 && experts <= 32) return launch_route<8, 4, false>(a, st);
    if (topk <= 16 && experts <= 64) return launch_route<16, 4, false>(a, st);
    if (experts <= 128) return launch_route<32, 4, false>(a, st);
    if (experts <= 256) return launch_route<64, 4, false>(a, st);
    if (experts <= 512) return launch_route<64, 8, false>(a, st);
    return launch_route<64, 16, false>(a, st);
}

extern "C" int mxl_topk_routing_bwd(const float* dprobs, const void* logits, int dtype, const int64_t* indices, int64_t tokens, int experts,
                                    int topk, int score, int renormalize, float scale, void* dlogits, void* stream) {
    if (!route_sizes_ok(tokens, experts, topk, dtype, score)) return MXL_EINVAL;
    if (tokens == 0) return MXL_OK;
    if (!dprobs || !logits || !indices || !dlogits) return MXL_EINVAL;
    if (!device_is_gfx950()) return MXL_ENODEV;
    RouteBwdArgs a{dprobs, logits, indices, dlogits, tokens, experts, topk, dtype, score == MXL_SCORE_SIGMOID, renormalize != 0, scale};
    if (score == MXL_SCORE_SIGMOID || renormalize) {
        if (topk <= 8 && experts <= 64 && tokens >= 8192) launch_route_bwd_chosen<8>(a, (hipStream_t)stream);
        else launch_route_bwd_chosen<32>(a, (hipStream_t)stream);
    } else {
        int64_t blocks = (tokens + RB_WAVES - 1) / RB_WAVES;
        if (blocks > 1024) blocks = 1024;
        hipLaunchKernelGGL(route_bwd_kernel, dim3((unsigned)blocks), dim3(RB_WAVES * 64), 0, (hipStream_t)stream, a);
    }
    return hipGetLastError() == hipSuccess ? MXL_OK : MXL_ELAUNCH;
}
