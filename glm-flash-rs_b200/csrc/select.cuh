// Selection of a row's experts by a rule: scores from logits, a bias that counts for the choice alone, groups of experts of which some
// stay, the top-k and their weights.
//
//   l = the logit, -inf where it is NaN;  s = 1 / (1 + exp(-l)) or exp(l - max) / sum exp(l - max)
//   c = s + bias (-inf where the bias is NaN);  without a bias c = l, whose order is that of the scores
//   value of a group = its largest c, or the sum of its two largest c (without a bias: s; +inf where one is); the largest groups stay, ties to
//   the lower one
//   choice = the topk largest c of the groups that stay, descending, ties to the lower id
//   weight = s * scale, or s / (sum of the chosen s) * scale, 0 where that sum is 0
// A softmax row whose largest logit is +inf shares 1 among its infinities (the limit); one without a logit above -inf has scores of 0.
// So every row gets topk different ids of the bank and finite weights, whatever is in it.
//
// Scores and sums are those of 64 bits: which of two is larger decides, and two that differ in the last place of 32 bits are no tie.  So that not
// every expert takes a 64-bit exponential, 32-bit values with known error bounds leave a few candidates, and those are ranked in 64 bits.
#pragma once
#include "common.cuh"

namespace gf {

struct SelRule {
    int softmax, groups, keep, top2, renorm;
    float scale;
};

// (value descending, id ascending): whether (a, i) comes before (b, j)
__device__ __forceinline__ bool sel_before(double a, int i, double b, int j) { return a > b || (a == b && i < j); }

__device__ __forceinline__ double sel_sigmoid(double l) { return 1. / (1. + exp(-l)); }

// One row by one warp in 64 bits throughout: whatever select_row leaves undecided.  c: E doubles of shared memory of this warp's (with a bias).
static __device__ __noinline__ void select_row_slowly(const float *row, const float *bias, int E, int topk, const SelRule &rule, double *c, int *picks,
                                               float *weights, int lane) {
    const unsigned all = 0xffffffffu;
    double top = 0., z = 1.;                             // softmax: the largest logit, the sum
    if (rule.softmax) {
        top = -INFINITY;
        for (int e = lane; e < E; e += 32) {
            const float l = row[e];
            if (l > top) top = l;
        }
        for (int m = 16; m; m >>= 1) top = fmax(top, __shfl_xor_sync(all, top, m));
        z = 0.;
        for (int e = lane; e < E; e += 32) {
            const float l = row[e];
            if (l == l && l > -INFINITY) z += l == top ? 1. : exp((double)l - top);
        }
        for (int m = 16; m; m >>= 1) z += __shfl_xor_sync(all, z, m);
    }
    auto score = [&](double l) {
        if (!rule.softmax) return sel_sigmoid(l);
        return l == -INFINITY ? 0. : l == top ? 1. / z : exp(l - top) / z;
    };
    auto logit = [&](int e) {
        const float f = row[e];
        return f == f ? (double)f : -INFINITY;
    };
    if (bias)
        for (int e = lane; e < E; e += 32) {
            const float b = bias[e];
            c[e] = b == b ? score(logit(e)) + (double)b : -INFINITY;
        }
    __syncwarp();
    auto value_of = [&](int e) { return bias ? c[e] : logit(e); };
    unsigned stay = all;
    const int per = E / rule.groups;
    if (rule.keep < rule.groups) {
        double value = -INFINITY;
        if (lane < rule.groups) {
            double first = -INFINITY, second = -INFINITY;
            for (int e = lane * per; e < (lane + 1) * per; ++e) {
                const double v = value_of(e);
                if (v > first) { second = first; first = v; }
                else if (v > second) second = v;
            }
            if (!rule.top2) value = first;
            else if (!bias) value = score(first) + (per > 1 ? score(second) : 0.);
            else value = per > 1 && first < INFINITY ? first + second : first;
        }
        int place = 0;
        for (int g = 0; g < rule.groups; ++g) place += sel_before(__shfl_sync(all, value, g), g, value, lane);
        stay = __ballot_sync(all, lane < rule.groups && place < rule.keep);
    }
    unsigned taken = 0;                                  // this lane's e = lane + 32 j
    double sum = 0., mine = 0.;
    for (int t = 0; t < topk; ++t) {
        double best = -INFINITY;
        int id = E;
        for (int e = lane, j = 0; e < E; e += 32, ++j)
            if (!(taken >> j & 1) && (stay >> (e / per) & 1)) {
                const double v = value_of(e);
                if (id == E || sel_before(v, e, best, id)) { best = v; id = e; }
            }
        for (int m = 16; m; m >>= 1) {
            const double ob = __shfl_xor_sync(all, best, m);
            const int oi = __shfl_xor_sync(all, id, m);
            if (oi < E && (id == E || sel_before(ob, oi, best, id))) { best = ob; id = oi; }
        }
        if ((id & 31) == lane) taken |= 1u << (id >> 5);
        const double s = score(logit(id));
        sum += s;
        if (lane == t) { mine = s; picks[t] = id; }
    }
    if (lane < topk) weights[lane] = (float)((rule.renorm ? (sum > 0. ? mine / sum : 0.) : mine) * rule.scale);
    if (lane == 0) { picks[topk] = E; weights[topk] = 1.f; }
}

// 32-bit values as integers of the same order
__device__ __forceinline__ unsigned sel_ordered(float v) {
    const unsigned u = __float_as_uint(v + 0.f);          // (-0 is 0)
    return u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float sel_value(unsigned o) { return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o); }

// How far off 32-bit values may be.  A sigmoid (fast exponential, 2 + 1.2 |x| units in the last place, times s (1 - s); fast quotient, 2 units): less
// than 2^-21.  A softmax score: less than 2^-18 of the largest possible one `most` (its sum: up to 37 additions one after another and the
// exponentials' own errors; x e^-x stays below 1/2).  c = s + bias by 2^-24 of itself in addition: together, since |bias| <= |c| + s, less than err (2
// most + |c|).
__device__ __forceinline__ float sel_err(bool softmax) { return softmax ? 1.f / (1 << 18) : 1.f / (1 << 21); }

// What few rows need, kept out of the others' way (registers):
// the sum of a softmax
__device__ __forceinline__ double sel_sum(const float *row, int E, float top, int lane) {
    double sum = 0.;
    for (int e = lane; e < E; e += 32) sum += exp((double)fmaxf(row[e], -INFINITY) - (double)top);
    for (int m = 16; m; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
    return sum;
}
// of the groups in `left` (the bits of their lanes, `wide` a group) how many come before this lane's, by their values in 64 bits
static __device__ __noinline__ int sel_groups_before(const float *row, const float *bias, int E, const SelRule &rule, float top, unsigned left, int wide, int lane) {
    const unsigned all = 0xffffffffu;
    const int per = E / rule.groups, g = lane / wide;
    // (without a bias a softmax's sum is left out: it scales all alike)
    const double sum64 = rule.softmax && bias ? sel_sum(row, E, top, lane) : 1.;
    auto score = [&](double l) { return rule.softmax ? exp(l - (double)top) / sum64 : sel_sigmoid(l); };
    double value = 0.;
    for (unsigned todo = left; todo;) {
        const int of = (__ffs(todo) - 1) / wide;
        todo &= ~(((1u << wide) - 1u) << of * wide);     // (two groups at least: wide <= 16)
        double one = -INFINITY, two = -INFINITY;
        for (int e = of * per + lane; e < (of + 1) * per; e += 32) {
            const double l = fmaxf(row[e], -INFINITY);
            double v = l;
            if (bias) {
                const float b = bias[e];
                v = b == b ? score(l) + (double)b : -INFINITY;
            }
            if (v > one) { two = one; one = v; }
            else if (v > two) two = v;
        }
        for (int m = 16; m; m >>= 1) {
            const double f = __shfl_xor_sync(all, one, m), t = __shfl_xor_sync(all, two, m);
            two = fmax(fmax(two, t), fmin(one, f));
            one = fmax(one, f);
        }
        const double sum = !rule.top2 ? one : !bias ? score(one) + (per > 1 ? score(two) : 0.) : per > 1 && one < INFINITY ? one + two : one;
        if (g == of) value = sum;
    }
    int before = 0;
    for (int i = 0; i < rule.groups; ++i) {
        const double other = __shfl_sync(all, value, i * wide);
        before += (left >> i * wide & 1) && sel_before(other, i, value, g);
    }
    return before;
}
// rank of this lane's candidate (logit l, bias b) among n by c in 64 bits
static __device__ __noinline__ int sel_rank(const float *row, int E, int softmax, float top, bool live, float l, float b, int id, int n, int lane) {
    const double sum64 = softmax ? sel_sum(row, E, top, lane) : 1.;
    double v = -INFINITY;
    if (live && b == b) v = (softmax ? exp((double)l - (double)top) / sum64 : sel_sigmoid(l)) + (double)b;
    int rank = 0;
    for (int i = 0; i < n; ++i) rank += sel_before(__shfl_sync(0xffffffffu, v, i), __shfl_sync(0xffffffffu, id, i), v, id);
    return rank;
}

// E values to shared memory, in flight on return.  All at once: through registers the loads of a loop wait for one
// another (800 clocks for every 32 experts), or the loop is unrolled.
__device__ __forceinline__ void sel_fetch(float *to, const float *from, int E, int lane) {
    const uint32_t at = smem_u32(to);
    if (((uintptr_t)from | E * 4) % 16 == 0)
        for (int e = 4 * lane; e < E; e += 128) asm volatile("cp.async.ca.shared.global [%0], [%1], 16;" ::"r"(at + 4 * e), "l"(from + e) : "memory");
    else
        for (int e = lane; e < E; e += 32) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(at + 4 * e), "l"(from + e) : "memory");
}

// behind the last expert
__device__ __forceinline__ void sel_pad(float *keys, int E, bool biased, int lane) {
    const int turns = (E + 31) >> 5, e = lane + 32 * (turns - 1);
    if (e >= E) {
        keys[e] = -INFINITY;
        if (biased) keys[32 * turns + e] = -INFINITY;
    }
}

// One row by one warp; E <= 1024, topk <= 31, groups <= 32.  keys: shared memory of this warp's, a multiple of 32 experts floats, as many again behind
// them with a bias; spot: 32 places.
//   1. 32-bit c of every expert, in shared memory (in registers the loops over them have to be unrolled: long code, fetched for one pass)
//   2. groups: 32-bit values by a few lanes a group; those that the error could carry over the border are valued in 64 bits by the whole warp
//   3. a lower bound of the topk-th largest c: of the largest values of the lanes' shares the topk-th; where that leaves more than 32, bisection
//   4. the candidates, those not provably below it, get a lane each: rank by comparison with all of them, in 64 bits if two are within the error
// 8192 rows of 288 experts in 8 groups 13.5 us, one row 3.4; selection one after another, all in 64 bits (select_row_slowly), 62 and 13.
// STAGED: keys (and biases) are there already, as sel_fetch and sel_pad leave them.
template <bool STAGED>
__device__ __forceinline__ void select_row(const float *row, const float *bias, int E, int topk, const SelRule &rule, float *keys, int2 *spot, int *picks,
                                           float *weights, int lane) {
    const unsigned all = 0xffffffffu;
    const bool exact = bias == nullptr, grouped = rule.keep < rule.groups;   // exact: the keys are the logits
    const float err = sel_err(rule.softmax);
    const int turns = (E + 31) >> 5;
    float *biases = keys + 32 * turns;
    float top = 0.f, z = 1.f, most = 1.f, mine = -INFINITY;                  // most: the largest score there can be;  mine: the lane's largest key
    bool sound = true;
    auto clean = [](float l) { return fmaxf(l, -INFINITY); };                // (NaN: -inf)
    // (fast exponential and reciprocal; 1 / inf is 0, as it should be)
    auto score = [&](float l) {
        if (rule.softmax) return __expf(l - top) * most;
        float r;
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + __expf(-l)));
        return r;
    };
    // every key of this lane by f(key, bias), four on their way at a time
    auto each = [&](bool biased, auto f) {
        float *p = keys + lane;
        const float *q = biases + lane;
        int j = 0;
        for (; j + 4 <= turns; j += 4, p += 128, q += 128) {
            float k[4], b[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                k[i] = p[32 * i];
                b[i] = biased ? q[32 * i] : 0.f;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) p[32 * i] = f(k[i], b[i]);
        }
        for (; j < turns; ++j, p += 32, q += 32) *p = f(*p, biased ? *q : 0.f);
    };
    if (!STAGED) {
        sel_fetch(keys, row, E, lane);
        if (!exact) sel_fetch(biases, bias, E, lane);
        sel_pad(keys, E, !exact, lane);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();
    if (rule.softmax) {
        each(false, [&](float l, float) {
            l = clean(l);
            mine = fmaxf(mine, l);
            return l;
        });
        top = sel_value(__reduce_max_sync(all, sel_ordered(mine)));
        z = 0.f;
        if (top - top == 0.f) {
            each(false, [&](float l, float) {
                z += expf(l - top);                      // (exp(-inf) is 0)
                return l;
            });
#pragma unroll
            for (int m = 16; m; m >>= 1) z += __shfl_xor_sync(all, z, m);
            most = 1.f / z;
        } else sound = false;                            // an infinity, or nothing
    }
    if (!exact) {
        mine = -INFINITY;
        each(true, [&](float l, float b) {
            l = clean(score(clean(l)) + b);
            mine = fmaxf(mine, l);
            return l;
        });
    } else if (!rule.softmax) {
        each(false, [&](float l, float) {
            l = clean(l);
            mine = fmaxf(mine, l);
            return l;
        });
    }
    __syncwarp();
    if (grouped) {
        const int per = E / rule.groups, wide = 32 >> (32 - __clz(rule.groups - 1)), g = lane / wide;    // lanes of a group
        float first = -INFINITY, second = -INFINITY;
        if (g < rule.groups)
#pragma unroll 4
            for (int e = lane - g * wide; e < per; e += wide) {
                const float v = keys[g * per + e];
                second = fmaxf(second, fminf(first, v));
                first = fmaxf(first, v);
            }
        const float own = first;
        for (int m = 1; m < wide; m <<= 1) {
            const float f = __shfl_xor_sync(all, first, m), s = __shfl_xor_sync(all, second, m);
            second = fmaxf(fmaxf(second, s), fminf(first, f));
            first = fmaxf(first, f);
        }
        float value = first;
        if (rule.top2 && exact) value = score(first) + (per > 1 ? score(second) : 0.f);
        else if (rule.top2 && per > 1 && first < INFINITY) value = first + second;
        const unsigned o = g < rule.groups ? sel_ordered(value) : 0u;
        int place = 0;
        for (int i = 0; i < rule.groups; ++i) {
            const unsigned other = __shfl_sync(all, o, i * wide);
            place += other > o || (other == o && i < g);
        }
        bool in = g < rule.groups && place < rule.keep;
        if (!(exact && !rule.top2)) {
            // Where the value may lie: c of the group's largest and second are off by err (2 most + |c|) each, however much of them cancels in the sum (without a
            // bias a sum of two scores, off by less).  Infinite terms are what they are; sums beyond the range are compared like infinities, and tie.
            const float terms = rule.top2 && !exact && per > 1 ? fabsf(first) + fabsf(second) : fabsf(value);
            const float off = terms < INFINITY ? 1.1f * err * (4.f * most + terms) : 0.f, low = value - off, high = value + off;
            const float worst = sel_value(__reduce_min_sync(all, in ? sel_ordered(low) : 0xffffffffu)),
                        best = sel_value(__reduce_max_sync(all, in || g >= rule.groups ? 0u : sel_ordered(high)));
            const bool open_question = g < rule.groups && !(in ? low > best : high < worst);
            unsigned left = __ballot_sync(all, open_question);
            if (left && sound) {
                const int places = rule.keep - __popc(__ballot_sync(all, in && !open_question && lane == g * wide));
                const int before = sel_groups_before(row, bias, E, rule, top, left, wide, lane);
                if (open_question) in = before < places;
            }
        }
        // experts of the other groups: NaN, which no comparison finds
        if (g < rule.groups && !in)
            for (int e = lane - g * wide; e < per; e += wide) keys[g * per + e] = NAN;
        __syncwarp();
        if (rule.keep * wide >= topk) mine = in ? own : -INFINITY;           // a lane's share of its group
        else {                                                               // too few lanes: every 32nd expert as before
            mine = -INFINITY;
            for (int e = lane; e < E; e += 32) mine = fmaxf(mine, keys[e]);
        }
    }
    // of the lanes' largest keys the topk-th
    unsigned bound = 0, rest = sel_ordered(mine);
    const unsigned highest = __reduce_max_sync(all, rest);
    for (int t = 0; t < topk; ++t) {
        bound = __reduce_max_sync(all, rest);
        const unsigned same = __ballot_sync(all, rest == bound);
        if (lane == __ffs(same) - 1) rest = 0;
    }
    auto threshold = [&](unsigned o) {
        const float t = sel_value(o);
        return exact || t - t != 0.f ? t : t - 2.5f * err * (2.f * most + fabsf(t));
    };
    // which keys of the lane are that large, a bit a turn
    auto marked = [&](float from) {
        unsigned mask = 0;
#pragma unroll 4
        for (int j = 0; j < turns; ++j) mask |= (unsigned)(keys[32 * j + lane] >= from) << j;
        if (lane + 32 * (turns - 1) >= E) mask &= ~(1u << (turns - 1));
        return mask;
    };
    auto count = [&](float from) { return (int)__reduce_add_sync(all, __popc(marked(from))); };
    unsigned mask = marked(threshold(bound));
    int n = (int)__reduce_add_sync(all, __popc(mask));
    if (n > 32) {                                        // (bound: at least topk are that large;  above: fewer)
        unsigned above = highest + 1;
        while (n > 32 && above - bound > 1) {
            const unsigned middle = bound + ((above - bound) >> 1);
            if (count(sel_value(middle)) >= topk) {
                bound = middle;
                n = count(threshold(bound));
            } else above = middle;
        }
        mask = marked(threshold(bound));
        if (n > 32 && exact) {                           // ties: the lowest ids of those at the bound
            mask = marked(sel_value(bound + 1));
            int left = topk - (int)__reduce_add_sync(all, __popc(mask));
            for (int j = 0; j < turns; ++j) {
                const unsigned same = __ballot_sync(all, lane + 32 * j < E && keys[32 * j + lane] == sel_value(bound));
                if ((same >> lane & 1) && __popc(same & ((1u << lane) - 1)) < left) mask |= 1u << j;
                left = max(left - __popc(same), 0);
            }
            n = topk;
        }
    }
    if (n <= 32) {                                       // a place for each
        int at = __popc(mask);
#pragma unroll
        for (int m = 1; m < 32; m <<= 1) {
            const int below = __shfl_up_sync(all, at, m);
            if (lane >= m) at += below;
        }
        at -= __popc(mask);
        for (; mask; mask &= mask - 1, ++at) {
            const int e = 32 * (__ffs(mask) - 1) + lane;
            spot[at] = make_int2(e, __float_as_int(keys[e]));
        }
    }
    if (n > 32) sound = false;                           // (ties within the error)
    if (sound) {
        __syncwarp();
        const bool live = lane < n;
        const int2 candidate = live ? spot[lane] : make_int2(E, 0);
        const int id = candidate.x;
        const float k32 = live ? __int_as_float(candidate.y) : -INFINITY, l = exact ? k32 : live ? clean(row[id]) : 0.f, apart = 2.f * err * (2.f * most + fabsf(k32));
        int rank = 0;
        bool close = false;
#pragma unroll 4
        for (int i = 0; i < n; ++i) {
            const int2 other = spot[i];
            const float k = __int_as_float(other.y);
            rank += k > k32 || (k == k32 && other.x < id);
            close |= other.x != id && !(fabsf(k - k32) > apart);
        }
        const float s = rule.softmax ? expf(l - top) * most : 1.f / (1.f + expf(-l));
        if (!exact && __any_sync(all, live && close)) {  // in 64 bits
            const float b = live ? bias[id] : 0.f;
            rank = sel_rank(row, E, rule.softmax, top, live, l, b, id, n, lane);
        }
        const bool chosen = live && rank < topk;
        float sum = chosen ? s : 0.f;
#pragma unroll
        for (int m = 16; m; m >>= 1) sum += __shfl_xor_sync(all, sum, m);
        if (rule.renorm && __any_sync(all, chosen && s < 1e-30f)) sound = false;       // (scores that 32 bits hold badly, or not at all)
        if (__all_sync(all, sound)) {
            if (chosen) {
                picks[rank] = id;
                weights[rank] = (rule.renorm ? __fdividef(s, sum) : s) * rule.scale;
            }
            if (lane == 0) { picks[topk] = E; weights[topk] = 1.f; }
            return;
        }
    }
    __syncwarp();
    select_row_slowly(row, bias, E, topk, rule, reinterpret_cast<double *>(keys), picks, weights, lane);
}

}  // namespace gf
