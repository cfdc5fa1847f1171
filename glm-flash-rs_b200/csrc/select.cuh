// Selection of a row's experts by a rule: scores from logits, a bias that counts for the choice alone, groups of experts of which some
// stay, the top-k and their weights.
//
//   l = the logit, -inf where it is NaN;  s = 1 / (1 + exp(-l)) or exp(l - max) / sum exp(l - max)
//   c = s + bias (-inf where the bias is NaN);  without a bias c = l, whose order is that of the scores
//   value of a group = its largest c, or the sum of its two largest c (without a bias: s); the largest groups stay, ties to the lower one
//   choice = the topk largest c of the groups that stay, descending, ties to the lower id
//   weight = s * scale, or s / (sum of the chosen s) * scale, 0 where that sum is 0
// A softmax row whose largest logit is +inf shares 1 among its infinities (the limit); one without a logit above -inf has scores of 0.
// So every row gets topk different ids of the bank and finite weights, whatever is in it.
//
// Scores and sums are those of 64 bits: which of two is larger decides, and two that differ in the last place of 32 bits are no tie.
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

// One row by one warp; E <= 1024, topk <= 31, groups <= 32.  c: E doubles of shared memory of this warp's.
__device__ __forceinline__ void select_row(const float *row, const float *bias, int E, int topk, const SelRule &rule, double *c, int *picks,
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
    for (int e = lane; e < E; e += 32) {
        const float f = row[e];
        const double l = f == f ? (double)f : -INFINITY;
        double v = l;
        if (bias) {
            const float b = bias[e];
            v = b == b ? score(l) + (double)b : -INFINITY;
        }
        c[e] = v;
    }
    __syncwarp();
    unsigned stay = all;
    const int per = E / rule.groups;
    if (rule.keep < rule.groups) {
        double value = -INFINITY;
        if (lane < rule.groups) {
            double first = -INFINITY, second = -INFINITY;
            for (int e = lane * per; e < (lane + 1) * per; ++e) {
                const double v = c[e];
                if (v > first) { second = first; first = v; }
                else if (v > second) second = v;
            }
            value = !rule.top2 ? first : bias ? (per > 1 ? first + second : first) : score(first) + (per > 1 ? score(second) : 0.);
        }
        int place = 0;
        for (int g = 0; g < rule.groups; ++g) place += sel_before(__shfl_sync(all, value, g), g, value, lane);
        stay = __ballot_sync(all, lane < rule.groups && place < rule.keep);
    }
    unsigned taken = 0;                                  // this lane's e = lane + 32 j
    double sum = 0.;
    double mine = 0.;
    for (int t = 0; t < topk; ++t) {
        double best = -INFINITY;
        int id = E;
        for (int e = lane, j = 0; e < E; e += 32, ++j)
            if (!(taken >> j & 1) && (stay >> (e / per) & 1) && (id == E || sel_before(c[e], e, best, id))) { best = c[e]; id = e; }
        for (int m = 16; m; m >>= 1) {
            const double ob = __shfl_xor_sync(all, best, m);
            const int oi = __shfl_xor_sync(all, id, m);
            if (oi < E && (id == E || sel_before(ob, oi, best, id))) { best = ob; id = oi; }
        }
        if ((id & 31) == lane) taken |= 1u << (id >> 5);
        const float f = row[id];
        const double s = score(f == f ? (double)f : -INFINITY);
        sum += s;
        if (lane == t) { mine = s; picks[t] = id; }
    }
    if (lane < topk) weights[lane] = (float)((rule.renorm ? (sum > 0. ? mine / sum : 0.) : mine) * rule.scale);
    if (lane == 0) { picks[topk] = E; weights[topk] = 1.f; }
}

}  // namespace gf
