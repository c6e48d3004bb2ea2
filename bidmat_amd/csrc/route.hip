// Routing of columns to experts: from a dense matrix of scores (experts x columns) to a sparse one of weights with topk
// nonzeros per column, and the gradient of the weights with respect to the scores.
//
//   p = softmax(z) or sigmoid(z) over a column's experts;   key = p + bias (z itself without bias and groups)
//   groups: the topgroups groups with the largest sum of their two largest keys stay open
//   the topk largest keys of the open groups are taken, the lower index first among equals; rows ascend in a column
//   weight = scale * p, or scale * p / (sum of the p that were taken)
//
// A score of -inf closes an expert to the column (a column of them is padding); where fewer than topk are open, the
// remaining entries name the lowest other experts with weight 0. A NaN among a column's scores makes its weights NaN.
//
// One wave per column. The groups are dealt to its lanes in order, a power of two of lanes to each, and a lane holds
// consecutive experts, so that the order of (lane, slot) is the order of the experts.
//
// What bounds it: not memory (a score is read once) but the instructions per column. The taken keys are found as
// a threshold: a count of the keys that reach a value is a compare per slot, the rest runs on the scalar unit, and the value
// that exactly topk keys reach takes about ten counts whatever topk is. Keys are compared in fp32 with a bound on their
// error; only a column with another key within that bound of the border is decided from keys in fp64 (take_exact).
// 256 experts in 8 groups, 65536 columns bf16, 8 taken: 43 us with 16 lanes per column, 200 vector and 46 scalar instructions
// per column (a wave per column 80 us; its bytes alone would take 8 us); 60 experts, 32768 columns fp32: 13 us, and 4 us to
// add up the counts; 512 experts, 32768 columns fp32: 34 us. Above 512 experts, or more than 16 taken, a wave per column: 1000
// experts, 16384 columns 48 us.
#include "columns.hpp"
#include "elems.hpp"
#include "kernels.hpp"
#include "workspace.hpp"
#include <limits.h>

namespace bm {
namespace {

constexpr float kLog2e = 1.44269504088896340736f;

struct Deal {            // how a column's experts lie in the lanes
    int lanes;           // lanes per group (a power of two)
    int size;            // experts per group
    int each;            // experts per lane
    int kp;              // topk rounded up to a power of two: lanes per column when the weights are written
    int batch;           // columns whose weights a wave writes together
    bool halves;         // 16 lanes per column: the open groups take at most eight of them
};

template <class V>
__device__ __forceinline__ V lanes_max(V x) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const V y = __shfl_xor(x, m, 64);
        x = y > x ? y : x;
    }
    return x;
}
// Reductions of the wave into a scalar register, and the inclusive prefix sum: shifts inside rows of 16 lanes, then row
// results broadcast onwards. On whole numbers each step is one instruction (a float maximum takes three).
#define BM_WAVE_STEPS(STEP) \
    STEP(0x111, 0xf) STEP(0x112, 0xf) STEP(0x114, 0xf) STEP(0x118, 0xf) /* row_shr 1, 2, 4, 8 */ \
    STEP(0x142, 0xa) STEP(0x143, 0xc)                                   /* row_bcast 15, 31 */
__device__ __forceinline__ int wave_max(int x) {
#define BM_STEP(ctrl, rows) x = max(x, __builtin_amdgcn_update_dpp(INT_MIN, x, ctrl, rows, 0xf, false));
    BM_WAVE_STEPS(BM_STEP)
#undef BM_STEP
    return __builtin_amdgcn_readlane(x, 63);
}
__device__ __forceinline__ int wave_min(int x) {
#define BM_STEP(ctrl, rows) x = min(x, __builtin_amdgcn_update_dpp(INT_MAX, x, ctrl, rows, 0xf, false));
    BM_WAVE_STEPS(BM_STEP)
#undef BM_STEP
    return __builtin_amdgcn_readlane(x, 63);
}
__device__ __forceinline__ int wave_prefix(int x) {
#define BM_STEP(ctrl, rows) x += __builtin_amdgcn_update_dpp(0, x, ctrl, rows, 0xf, false);
    BM_WAVE_STEPS(BM_STEP)
#undef BM_STEP
    return x;
}
__device__ __forceinline__ float wave_sum(float x) {
#define BM_STEP(ctrl, rows) x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), ctrl, rows, 0xf, false));
    BM_WAVE_STEPS(BM_STEP)
#undef BM_STEP
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}

// Floats as whole numbers of the same order (and back: the map is its own inverse), -0 as 0. kShut stands below all of them.
constexpr int kShut = INT_MIN;
__device__ __forceinline__ int flip(int i) { return i ^ ((i >> 31) & 0x7fffffff); }
__device__ __forceinline__ int ordered(float x) { return flip(__float_as_int(x + 0.f)); }
__device__ __forceinline__ float number(int i) { return __int_as_float(flip(i)); }

// Which of a column's experts are taken, from keys in 64 bits: bit j of the result is this lane's slot j. Rarely called: a
// function of its own that reads its scores again (zp: of this lane's first expert), keeps its keys in LDS (slot j of lane
// l at key[64 * j + l]) and unrolls nothing, so that the loop around it keeps its registers (119 with all of it inline).
template <class T>
__device__ __noinline__ unsigned take_exact(const T* zp, const float* bias, double* key, int own, int each, int kind, int ngroups,
                                            int topgroups, int topk, int lanes) {
    const double ninf = -__builtin_inf();
    const int l = threadIdx.x & 63;
    key += l;
    const bool plain = bias == nullptr && ngroups == 1, softmax = kind == 0 && !plain;
    double top = ninf, sum = 0.;
    if (softmax) {
#pragma unroll 1
        for (int j = 0; j < own; ++j) top = fmax(top, (double)(float)zp[j]);
        top = lanes_max(top);
    }
#pragma unroll 1
    for (int j = 0; j < each; ++j) {
        const double z = j < own ? (double)(float)zp[j] : ninf;
        double k = z;
        if (!plain) {
            const double e = z > ninf ? exp(softmax ? z - top : -z) : 0.;
            k = softmax ? e : 1. / (1. + e);
            sum += e;
            if (!softmax && bias != nullptr && j < own) k += (double)bias[j];
        }
        key[64 * j] = z > ninf && k > ninf ? k : ninf;
    }
    if (softmax) {
        for (int m = 1; m < 64; m <<= 1) sum += __shfl_xor(sum, m, 64);
#pragma unroll 1
        for (int j = 0; j < own; ++j) {
            double k = key[64 * j];
            if (!(k > ninf)) continue;
            k = k / sum + (bias != nullptr ? (double)bias[j] : 0.);
            key[64 * j] = k > ninf ? k : ninf;
        }
    }
    bool shut = false;
    if (ngroups > 1) {
        double best = ninf, second = ninf;
#pragma unroll 1
        for (int j = 0; j < each; ++j) {
            const double k = key[64 * j], low = k < best ? k : best;
            second = low > second ? low : second;
            best = k > best ? k : best;
        }
        for (int m = 1; m < lanes; m <<= 1) {
            const double ob = __shfl_xor(best, m, 64), os = __shfl_xor(second, m, 64);
            const double low = ob < best ? ob : best, high = os > second ? os : second;
            second = low > high ? low : high;
            best = ob > best ? ob : best;
        }
        const double mine = second > ninf ? best + second : best;
        const int g = l / lanes;
        int before = 0;
#pragma unroll 1
        for (int q = 0; q < ngroups; ++q) {
            const double other = __shfl(mine, q * lanes, 64);
            before += other > mine || (other == mine && q < g);
        }
        shut = before >= topgroups;
    }
    unsigned taken = 0;
#pragma unroll 1
    for (int r = 0; r < topk; ++r) {
        double best = ninf;
        int at = 0;
#pragma unroll 1
        for (int j = 0; j < each; ++j) {
            const double k = key[64 * j];
            if (!shut && !(taken >> j & 1) && k > best) { best = k; at = j; }
        }
        const double top1 = lanes_max(best);
        if (!(top1 > ninf)) break;
        if (l == __builtin_ctzll(__ballot(best == top1))) taken |= 1u << at;
    }
    return taken;
}

template <int N>
__device__ __forceinline__ int count_from(const int (&key)[N], int t) {
    int c = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) c += __popcll(__ballot(key[j] >= t));
    return c;
}

// The border below the `want` largest of the wave's keys, of which more than want are open: they are the keys >= t, and
// where ties > 0 only the first `ties` of those that equal t.
struct Border { int t, ties; };
template <int N>
__device__ __forceinline__ Border find_border(const int (&key)[N], int want) {
    int best = key[0];
#pragma unroll
    for (int j = 1; j < N; ++j) best = max(best, key[j]);
    int hi = wave_max(best) + 1, over = 0;
    // the least of the lanes' largest keys is reached by at least as many keys as lanes have an open one
    int lo = wave_min(best == kShut ? INT_MAX : best);
    int n = count_from(key, lo);
    if (N > 1 && n < want) {
        int least = INT_MAX;
#pragma unroll
        for (int j = 0; j < N; ++j) least = min(least, key[j] == kShut ? INT_MAX : key[j]);
        lo = wave_min(least);
        n = count_from(key, lo);
    }
    while (n != want && (unsigned)hi - (unsigned)lo > 1u) {
        const int mid = lo + (int)(((unsigned)hi - (unsigned)lo) >> 1);
        const int c = count_from(key, mid);
        if (c >= want) { lo = mid; n = c; } else { hi = mid; over = c; }
    }
    return {lo, n > want ? want - over : 0};
}
// Whether keys that are off by at most e each have the same largest `want` as the exact ones.
template <int N>
__device__ __forceinline__ bool border_clear(const int (&key)[N], const Border& b, int want, float e) {
    const float t = number(b.t);
    return b.ties == 0 && count_from(key, wave_uniform(ordered(t + e))) == want && count_from(key, wave_uniform(ordered(t - e))) == want;
}

// The same in fp32; false: some key lies too close to a border.
template <class T, int VPL>
__device__ __forceinline__ bool take_fast(const RouteArgs& a, const Deal& d, const float (&z)[VPL], const float (&bias)[VPL], float bmax,
                                          float top, float by, unsigned& taken) {
    const int l = threadIdx.x & 63;
    int key[VPL];
    const bool plain = a.bias == nullptr && a.ngroups == 1;
    if (plain) {
        // scores of 16 bits differ in their upper bits only: fewer halvings until two that are equal are told so
        constexpr int shift = sizeof(T) == 4 ? 0 : __is_same(T, f16_t) ? 13 : 16;
#pragma unroll
        for (int j = 0; j < VPL; ++j) key[j] = z[j] > -INFINITY ? ordered(z[j]) >> shift : kShut;
    } else {
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
            float p;
            if (a.kind == 0) p = __builtin_amdgcn_exp2f((z[j] - top) * kLog2e) * by;
            else p = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-z[j] * kLog2e));
            p += bias[j];
            key[j] = z[j] > -INFINITY && p > -INFINITY ? ordered(p) : kShut;
        }
    }
    // Error of a key near the value v: p = key - bias is off by up to 2^-16 of itself (exp of an argument of up to 88, the
    // sum), a sigmoid also by less than 2^-20 at all.
    const float most = a.kind == 0 ? INFINITY : 0x1p-20f * (1.f + bmax);
    if (a.ngroups > 1) {
        int best = key[0], second = kShut;
#pragma unroll
        for (int j = 1; j < VPL; ++j) {
            second = max(second, min(best, key[j]));
            best = max(best, key[j]);
        }
        auto merge = [&](int ob, int os) {
            second = max(min(best, ob), max(second, os));
            best = max(best, ob);
        };
#define BM_MERGE(ctrl) merge(__builtin_amdgcn_update_dpp(0, best, ctrl, 0xf, 0xf, false), __builtin_amdgcn_update_dpp(0, second, ctrl, 0xf, 0xf, false))
        if (d.lanes >= 2) BM_MERGE(DPP_QUAD_XOR1);
        if (d.lanes >= 4) BM_MERGE(DPP_QUAD_XOR2);
        if (d.lanes >= 8) BM_MERGE(DPP_ROW_HALF_MIRROR);
        if (d.lanes >= 16) BM_MERGE(DPP_ROW_MIRROR);
        if (d.lanes >= 32) merge(__shfl_xor(best, 16, 64), __shfl_xor(second, 16, 64));
#undef BM_MERGE
        const int mine = best == kShut ? kShut : ordered(second == kShut ? number(best) : number(best) + number(second));
        // one lane of each group stands for it
        const int score[1] = {(l & (d.lanes - 1)) == 0 ? mine : kShut};
        if (__popcll(__ballot(score[0] != kShut)) > a.topgroups) {
            const Border b = find_border(score, a.topgroups);
            if (!border_clear(score, b, a.topgroups, fminf(2.f * most, 0x1p-15f * (fabsf(number(b.t)) + 2.f * bmax)))) return false;
            const bool shut = mine < b.t;
#pragma unroll
            for (int j = 0; j < VPL; ++j) key[j] = shut ? kShut : key[j];
        }
    }
    taken = 0;
    int open = 0;
#pragma unroll
    for (int j = 0; j < VPL; ++j) open += __popcll(__ballot(key[j] != kShut));
    if (open <= a.topk) {
#pragma unroll
        for (int j = 0; j < VPL; ++j) taken |= key[j] != kShut ? 1u << j : 0u;
        return true;
    }
    const Border b = find_border(key, a.topk);
    if (!plain && !border_clear(key, b, a.topk, fminf(most, 0x1p-16f * (fabsf(number(b.t)) + bmax)))) return false;
#pragma unroll
    for (int j = 0; j < VPL; ++j) taken |= key[j] >= b.t ? 1u << j : 0u;
    if (b.ties > 0) {
        // exact keys: of those that equal the border the first ones stay
        unsigned equal = 0;
#pragma unroll
        for (int j = 0; j < VPL; ++j) equal |= key[j] == b.t ? 1u << j : 0u;
        int left = b.ties - (wave_prefix(__popc(equal)) - __popc(equal));
        for (; equal != 0; equal &= equal - 1)
            if (left-- <= 0) taken &= ~(equal & -equal);
    }
    return true;
}

// Sum / largest over aligned groups of n lanes, n a power of two known at run time (steps of group_allsum).
__device__ __forceinline__ float lanes_sum_rt(float x, int n) {
    if (n >= 2) x += dpp_mov<DPP_QUAD_XOR1>(x);
    if (n >= 4) x += dpp_mov<DPP_QUAD_XOR2>(x);
    if (n >= 8) x += dpp_mov<DPP_ROW_HALF_MIRROR>(x);
    if (n >= 16) x += dpp_mov<DPP_ROW_MIRROR>(x);
    if (n >= 32) x += __shfl_xor(x, 16, 64);
    if (n >= 64) x += __shfl_xor(x, 32, 64);
    return x;
}
__device__ __forceinline__ float lanes_max_rt(float x, int n) {
    if (n >= 2) x = fmaxf(x, dpp_mov<DPP_QUAD_XOR1>(x));
    if (n >= 4) x = fmaxf(x, dpp_mov<DPP_QUAD_XOR2>(x));
    if (n >= 8) x = fmaxf(x, dpp_mov<DPP_ROW_HALF_MIRROR>(x));
    if (n >= 16) x = fmaxf(x, dpp_mov<DPP_ROW_MIRROR>(x));
    if (n >= 32) x = fmaxf(x, __shfl_xor(x, 16, 64));
    if (n >= 64) x = fmaxf(x, __shfl_xor(x, 32, 64));
    return x;
}
// Of the weights: expf and divisions, right to a few units however far a score lies below the largest (the hardware's exponential
// of x * log2(e) is off by |x| units, and saves nothing: 256 experts x 65536 columns 42.3 us, with these 42.2; 60 x 32768 14.3, 14.4).
__device__ __forceinline__ float sigmoid_of(float x) { return 1.f / (1.f + expf(-x)); }

constexpr int kRouteBatch = 8;           // columns whose weights one wave writes together, at most
struct Chosen {                          // of one wave
    unsigned short row[kRouteBatch][kRouteMaxTop];      // bit 15: named only to fill the column, weight 0
    float top[kRouteBatch], by[kRouteBatch];            // softmax over all: p = exp(z - top) * by; top NaN: the column holds one
};

// The weights, rows and counts of columns c0 .. c0 + cols - 1, whose experts lie in ch: kp lanes per column.
template <class T>
__device__ __forceinline__ void write_weights(const RouteArgs& a, const Deal& d, const Chosen& ch, long long c0, int cols, int* hist) {
    const int l = threadIdx.x & 63;
    for (int b0 = 0; b0 < cols; b0 += 64 / d.kp) {
        const int b = b0 + l / d.kp, s = l & (d.kp - 1);
        const bool on = b < cols && s < a.topk;
        const int e = on ? ch.row[b][s] : 0x8000, r = e & 0x7fff;
        const bool valid = on && e < 0x8000;
        const float top = b < cols ? ch.top[b] : 0.f, by = b < cols ? ch.by[b] : 0.f;
        const long long c = c0 + b;
        const float z = valid ? (float)((const T*)a.Z)[c * a.ldz + r] : -INFINITY;
        float p;
        if (a.renorm) {
            const float high = lanes_max_rt(z, d.kp);
            // Far below 0 sigmoid(z) is exp(z) to within a factor 1 + exp(z): with all taken scores below -30 their
            // shares are a softmax's, where the sigmoids themselves may have left the range of fp32.
            p = a.kind == 0 || high < -30.f ? expf(z - high) : sigmoid_of(z);
            p = valid ? p : 0.f;
            const float sum = lanes_sum_rt(p, d.kp);
            p = sum > 0.f ? a.scale * (p / sum) : 0.f;          // (scale / sum may leave fp32)
        } else {
            p = a.scale * (a.kind == 0 ? expf(z - top) * by : sigmoid_of(z));
            p = valid ? p : 0.f;
        }
        if (on) {
            const long long q = c * a.topk + s;
            a.ir[q] = r;
            a.data[q] = top != top ? NAN : p;
            if (a.ic != nullptr) a.ic[q] = (int)c;
            if (valid && a.counts != nullptr) atomicAdd(&hist[r], 1);
            if (s == 0 && a.jc != nullptr) {
                a.jc[c] = (int)(c * a.topk);
                if (c == a.ncols - 1) a.jc[c + 1] = (int)((c + 1) * a.topk);
            }
        }
    }
}

// BLOCK threads; ONE: a single workgroup, which writes the counts; otherwise each workgroup its share of them.
template <class T, int VPL, int BLOCK, bool ONE>
__global__ __launch_bounds__(BLOCK) void k_route(RouteArgs a, Deal d, int* shares) {
    constexpr int WAVES = BLOCK / 64;
    __shared__ int hist[kRouteMaxExperts];
    __shared__ Chosen chosen[WAVES];
    extern __shared__ double exact_keys[];      // 64 * d.each per wave
    if (a.counts != nullptr) {
        for (int e = threadIdx.x; e < a.nexperts; e += BLOCK) hist[e] = 0;
        __syncthreads();
    }
    const int l = threadIdx.x & 63, wave = wave_uniform(threadIdx.x >> 6);
    Chosen& ch = chosen[wave];
    const int g = l / d.lanes, o = (l & (d.lanes - 1)) * d.each;       // group of this lane, first slot inside it
    const int first = g * d.size + o;
    const int room = d.size - o < d.each ? d.size - o : d.each;
    const int own = g < a.ngroups && room > 0 ? room : 0;              // experts of this lane
    float bias[VPL];
    int most_bias = 0;          // a NaN stands above infinity here
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
        bias[j] = a.bias != nullptr && j < own ? a.bias[first + j] : 0.f;
        most_bias = max(most_bias, __float_as_int(bias[j]) & 0x7fffffff);
    }
    const float bmax = __int_as_float(wave_max(most_bias));
    const bool exact_only = !(bmax < 0x1p100f);          // the error bounds below are for finite biases
    const bool sums = a.kind == 0 && (a.bias != nullptr || a.ngroups > 1 || !a.renorm);      // softmax over all is needed
    const long long end = (a.ncols - 1LL) * a.ldz + a.nexperts;                              // of the matrix, in elements
    const long long step = (long long)gridDim.x * WAVES * d.batch;
    for (long long c0 = ((long long)blockIdx.x * WAVES + wave) * d.batch; c0 < a.ncols; c0 += step) {
        const int cols = (int)(a.ncols - c0 < d.batch ? a.ncols - c0 : d.batch);
        for (int b = 0; b < cols; ++b) {
            const long long at = (c0 + b) * a.ldz + first;
            float z[VPL];
            if (VPL >= 2 && at + VPL <= end) {          // wide loads may run into the next column, not out of the matrix
                T raw[VPL];
                __builtin_memcpy(raw, (const T*)a.Z + at, sizeof(raw));
#pragma unroll
                for (int j = 0; j < VPL; ++j) z[j] = j < own ? (float)raw[j] : -INFINITY;
            } else {
#pragma unroll
                for (int j = 0; j < VPL; ++j) z[j] = j < own ? (float)((const T*)a.Z)[at + j] : -INFINITY;
            }
            // a NaN, or +inf where the softmax has no value
            const int odd_class = a.kind == 0 ? 0x203 : 0x003;
            bool odd = false;
#pragma unroll
            for (int j = 0; j < VPL; ++j) odd = odd || __builtin_amdgcn_classf(z[j], odd_class);
            const bool bad = __ballot(odd) != 0;
            float top = 0.f, by = 1.f;
            if (sums) {
                top = z[0];
#pragma unroll
                for (int j = 1; j < VPL; ++j) top = fmaxf(top, z[j]);
                top = number(wave_max(ordered(top)));
                float sum = 0.f;
#pragma unroll
                for (int j = 0; j < VPL; ++j) sum += z[j] > -INFINITY ? __builtin_amdgcn_exp2f((z[j] - top) * kLog2e) : 0.f;
                sum = wave_sum(sum);
                by = sum > 0.f ? 1.f / sum : 0.f;
            }
            unsigned taken = 0;
            if (!bad && (exact_only || !take_fast<T, VPL>(a, d, z, bias, bmax, top, by, taken)))
                taken = take_exact<T>((const T*)a.Z + at, a.bias != nullptr ? a.bias + first : nullptr, exact_keys + wave * 64 * d.each, own,
                                      d.each, a.kind, a.ngroups, a.topgroups, a.topk, d.lanes);
            // fewer than topk open: the lowest others fill the column
            const unsigned valid = taken;
            int upto = wave_prefix(__popc(taken));
            const int have = __builtin_amdgcn_readlane(upto, 63);
            if (have < a.topk) {
                unsigned rest = own > 0 ? ~taken & (own >= 32 ? ~0u : (1u << own) - 1u) : 0u;
                int left = a.topk - have - (wave_prefix(__popc(rest)) - __popc(rest));
                for (; rest != 0 && left > 0; rest &= rest - 1, --left) taken |= rest & -rest;
                upto = wave_prefix(__popc(taken));
            }
            int before = upto - __popc(taken);
            for (unsigned t = taken; t != 0; t &= t - 1) {
                const int j = __builtin_ctz(t);
                ch.row[b][before++] = (unsigned short)((first + j) | (valid >> j & 1 ? 0 : 0x8000));
            }
            if (l == 0) {
                ch.top[b] = bad ? NAN : top;
                ch.by[b] = by;
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        write_weights<T>(a, d, ch, c0, cols, hist);
        __builtin_amdgcn_wave_barrier();
    }
    if (a.counts != nullptr) {
        __syncthreads();
        for (int e = threadIdx.x; e < a.nexperts; e += BLOCK) {
            if (ONE) a.counts[e] = hist[e];
            else shares[(size_t)blockIdx.x * a.nexperts + e] = hist[e];
        }
    }
}

// One column decided from keys in 64 bits by a whole wave; its experts (bit 15: named only to fill the column) go to out.
template <class T>
__device__ __forceinline__ void exact_column(const RouteArgs& a, const Deal& d, long long c, double* keys, unsigned short* out) {
    const int l = threadIdx.x & 63, g = l / d.lanes, o = (l & (d.lanes - 1)) * d.each;
    const int first = g * d.size + o, room = d.size - o < d.each ? d.size - o : d.each;
    const int own = g < a.ngroups && room > 0 ? room : 0;
    const unsigned valid = take_exact<T>((const T*)a.Z + c * a.ldz + first, a.bias != nullptr ? a.bias + first : nullptr, keys, own, d.each,
                                         a.kind, a.ngroups, a.topgroups, a.topk, d.lanes);
    unsigned taken = valid;
    int upto = wave_prefix(__popc(taken));
    const int have = __builtin_amdgcn_readlane(upto, 63);
    if (have < a.topk) {
        unsigned rest = own > 0 ? ~taken & (own >= 32 ? ~0u : (1u << own) - 1u) : 0u;
        int left = a.topk - have - (wave_prefix(__popc(rest)) - __popc(rest));
        for (; rest != 0 && left > 0; rest &= rest - 1, --left) taken |= rest & -rest;
        upto = wave_prefix(__popc(taken));
    }
    int before = upto - __popc(taken);
    for (unsigned t = taken; t != 0; t &= t - 1) {
        const int j = __builtin_ctz(t);
        out[before++] = (unsigned short)((first + j) | (valid >> j & 1 ? 0 : 0x8000));
    }
}

// ---- 16 lanes per column
// The same for up to 512 experts in up to 16 groups and up to 16 of them taken: four columns per wave, so that what lanes do
// together costs a quarter per column and needs no step across rows of 16 lanes. A lane holds up to 32 experts; counts
// run on the vector unit (a compare and an addition per slot).
template <int CTRL>
__device__ __forceinline__ int row_move(int x) { return __builtin_amdgcn_update_dpp(0, x, CTRL, 0xf, 0xf, true); }
#define BM_ROW_ALL(x, op)                                                     \
    x = op(x, row_move<DPP_QUAD_XOR1>(x)); x = op(x, row_move<DPP_QUAD_XOR2>(x)); \
    x = op(x, row_move<DPP_ROW_HALF_MIRROR>(x)); x = op(x, row_move<DPP_ROW_MIRROR>(x))
__device__ __forceinline__ int middle(int x, int y, int z) {
    int r;
    asm("v_med3_i32 %0, %1, %2, %3" : "=v"(r) : "v"(x), "v"(y), "v"(z));
    return r;
}
__device__ __forceinline__ int add_int(int x, int y) { return x + y; }
__device__ __forceinline__ int row_max(int x) { BM_ROW_ALL(x, max); return x; }
__device__ __forceinline__ int row_min(int x) { BM_ROW_ALL(x, min); return x; }
__device__ __forceinline__ int row_sum(int x) { BM_ROW_ALL(x, add_int); return x; }
__device__ __forceinline__ int row_prefix(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    return x;
}
template <int N>
__device__ __forceinline__ int row_count(const int (&key)[N], int t) {
    int c = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) c += key[j] >= t;
    return row_sum(c);
}

// Distance from lo to the smallest key of the column that reaches it.
template <int N>
__device__ __forceinline__ unsigned row_least_from(const int (&key)[N], int lo) {
    unsigned x = ~0u;
#pragma unroll
    for (int j = 0; j < N; ++j) x = min(x, (unsigned)key[j] - (unsigned)lo);
#define BM_MIN(ctrl) x = min(x, (unsigned)row_move<ctrl>((int)x))
    BM_MIN(DPP_QUAD_XOR1); BM_MIN(DPP_QUAD_XOR2); BM_MIN(DPP_ROW_HALF_MIRROR); BM_MIN(DPP_ROW_MIRROR);
#undef BM_MIN
    return x;
}

// How many groups' scores lie at or above lo, and above hi, among the other groups of the column (LG lanes per group).
template <int LG, int N>
__device__ __forceinline__ void row_rank(float score, float lo, float hi, int& reach, int& pass) {
    if constexpr (N < 16) {
        if constexpr (N % LG == 0) {
            const float other = __int_as_float(row_move<0x120 + N>(__float_as_int(score)));      // row_ror N
            reach += other >= lo;
            pass += other > hi;
        }
        row_rank<LG, N + 1>(score, lo, hi, reach, pass);
    }
}

// How many of the other lanes of the column hold a larger key.
template <int N>
__device__ __forceinline__ void row_before(int key, int& before) {
    if constexpr (N < 16) {
        before += row_move<0x120 + N>(key) > key;      // row_ror N
        row_before<N + 1>(key, before);
    }
}

// Scores as keys: those of 16 bits get the expert's number into their lower bits, so that no two are equal and the lower
// expert stands higher. score_key: the lowest key that a score of at least x can have.
template <class T> constexpr int kScoreShift = sizeof(T) == 4 ? 0 : __is_same(T, f16_t) ? 13 : 16;
template <class T>
__device__ __forceinline__ float key_score(int key) {
    if constexpr (sizeof(T) == 4) return number(key);
    const int o = (int)((unsigned)(key >> 9) << kScoreShift<T>);
    return number(o < 0 ? o | ((1 << kScoreShift<T>) - 1) : o);
}
template <class T>
__device__ __forceinline__ int score_key(float x) {
    const int o = ordered(x);
    if constexpr (sizeof(T) == 4) return o;
    return ((o < 0 ? o : o + (1 << kScoreShift<T>) - 1) >> kScoreShift<T>) * 512;
}

// Without a bias the scores themselves are compared: p rises with them. Other keys are p + bias + bmax: never negative, so that
// their bits are in order as they are. Returns the taken slots; fine = false where a key lies too close to a border.
template <class T, int VPL>
__device__ __forceinline__ unsigned take_row(const RouteArgs& a, const Deal& d, const float (&z)[VPL], const float (&bias)[VPL], float bmax,
                                             float top, float by, int first, bool shut, int* sixteen, bool& fine) {
    const bool direct = a.bias == nullptr;
    int key[VPL];
    if (direct) {
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
            int k = ordered(z[j]);
            if constexpr (sizeof(T) == 2) k = (int)((unsigned)(k >> kScoreShift<T>) << 9) | (511 - first - j);
            key[j] = z[j] > -INFINITY ? k : kShut;
        }
    } else {
        if (a.kind == 0) {
#pragma unroll
            for (int j = 0; j < VPL; ++j) key[j] = __float_as_int(__builtin_amdgcn_exp2f((z[j] - top) * kLog2e) * by + bias[j]);
        } else {
#pragma unroll
            for (int j = 0; j < VPL; ++j) key[j] = __float_as_int(__builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-z[j] * kLog2e)) + bias[j]);
        }
        if (shut) {
#pragma unroll
            for (int j = 0; j < VPL; ++j) key[j] = z[j] > -INFINITY ? key[j] : kShut;
        }
    }
    // Error of a key: p is off by up to 2^-16 of itself (exp of an argument of up to 88, the sum; by is the largest p of a
    // softmax), a sigmoid by less than 2^-21 at all; the additions of bias and bmax by 2^-23 of the result.
    const float most = a.kind == 0 ? 0x1p-16f * by + 0x1p-21f * (by + bmax) : 0x1p-20f * (1.f + 3.f * bmax);
    int best = key[0], second = kShut;
#pragma unroll
    for (int j = 1; j < VPL; ++j) {
        second = middle(second, best, key[j]);
        best = max(best, key[j]);
    }
    fine = true;
    if (a.ngroups > 1) {
        int b1 = best, b2 = second;
        auto merge = [&](int ob, int os) {
            b2 = max(min(b1, ob), max(b2, os));
            b1 = max(b1, ob);
        };
        if (d.lanes >= 2) merge(row_move<DPP_QUAD_XOR1>(b1), row_move<DPP_QUAD_XOR1>(b2));
        if (d.lanes >= 4) merge(row_move<DPP_QUAD_XOR2>(b1), row_move<DPP_QUAD_XOR2>(b2));
        if (d.lanes >= 8) merge(row_move<DPP_ROW_HALF_MIRROR>(b1), row_move<DPP_ROW_HALF_MIRROR>(b2));
        float p1 = __int_as_float(b1), p2 = __int_as_float(b2);
        if (direct) {
            const float z1 = key_score<T>(b1), z2 = key_score<T>(b2);
            p1 = a.kind == 0 ? __builtin_amdgcn_exp2f((z1 - top) * kLog2e) * by : __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-z1 * kLog2e));
            p2 = a.kind == 0 ? __builtin_amdgcn_exp2f((z2 - top) * kLog2e) * by : __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-z2 * kLog2e));
        }
        // each key carries bmax once: a group with a single open expert gets its second one here
        const float score = b1 == kShut ? -INFINITY : p1 + (b2 == kShut ? bmax : p2);
        const float e = 2.f * fminf(2.f * most + 0x1p-22f * score, 0x1p-14f * score);
        int reach = 0, pass = 0;
        switch (d.lanes) {
        case 1: row_rank<1, 1>(score, score - e, score + e, reach, pass); break;
        case 2: row_rank<2, 1>(score, score - e, score + e, reach, pass); break;
        case 4: row_rank<4, 1>(score, score - e, score + e, reach, pass); break;
        default: row_rank<8, 1>(score, score - e, score + e, reach, pass); break;
        }
        const bool in = reach < a.topgroups, out = pass >= a.topgroups;
        if (b1 != kShut && !in && !out) fine = false;
        if (!in || b1 == kShut) {
            best = second = kShut;
#pragma unroll
            for (int j = 0; j < VPL; ++j) key[j] = kShut;
        }
    }
    const int want = a.topk;
    // [lo, hi): the border's bracket; n keys reach lo. First among the lanes' two largest, where want keys exist there.
    int lo, hi = row_max(best), n;
    hi = hi == kShut ? kShut + 2 : hi + 1;
    {
        bool enough;
        if (d.halves) {
            // at most eight lanes are open: their two largest keys fit the sixteen lanes, one each
            const bool mine = best != kShut;
            const int i = threadIdx.x & 15, at = row_prefix(mine) - 1;
            sixteen[i] = kShut;
            __builtin_amdgcn_wave_barrier();          // a wave's LDS operations take effect in order
            if (mine && at < 8) {
                sixteen[at] = best;
                sixteen[8 + at] = second;
            }
            __builtin_amdgcn_wave_barrier();
            const int key16 = sixteen[i];
            int before = 0;
            row_before<1>(key16, before);
            enough = row_sum(key16 != kShut) >= want;
            lo = row_min(before < want && key16 != kShut ? key16 : INT_MAX);
        } else if (__ballot(row_sum(best != kShut) < 2 * want) == 0) {
            // open keys in twice as many lanes as keys are wanted: few lanes hold two of them, so that the want-th of the lanes'
            // largest keys is close to the border, and on its far side
            int before = 0;
            row_before<1>(best, before);
            lo = row_min(before < want && best != kShut ? best : INT_MAX);
            enough = true;
        } else {
            const int two[2] = {best, second};
            int end = hi;
            lo = row_min(second == kShut ? (best == kShut ? INT_MAX : best) : second);
            n = row_count(two, lo);
            enough = n >= want;
            while (__ballot(enough && n != want && (unsigned)end - (unsigned)lo > 1u) != 0) {
                const int mid = lo + (int)(((unsigned)end - (unsigned)lo) >> 1);
                const int m = row_count(two, mid);
                if (enough) {
                    if (m >= want) { lo = mid; n = m; } else end = mid;
                }
            }
        }
        if (__ballot(!enough) != 0) {
            int least = INT_MAX;
#pragma unroll
            for (int j = 0; j < VPL; ++j) least = min(least, key[j] == kShut ? INT_MAX : key[j]);
            least = row_min(least);
            lo = enough ? lo : least;
        }
        n = row_count(key, lo);
    }
    while (__ballot(n > want) != 0) {
        const bool wide = (unsigned)hi - (unsigned)lo > 1u;
        if (__ballot(n > want + 3 && wide) != 0) {
            const int mid = lo + (int)(((unsigned)hi - (unsigned)lo) >> 1);
            const int m = row_count(key, mid);
            if (m >= want) { lo = n > want ? mid : lo; n = n > want ? m : n; } else hi = n > want ? mid : hi;
        } else {
            // the smallest key of those that reach lo goes; equal ones are found out at the end
            const int next = lo + (int)row_least_from(key, lo) + 1;
            if (n > want) {
                if (!wide) fine = false;
                lo = wide ? next : lo;
                n = wide ? n - 1 : want;
            }
        }
    }
    if (n > 0) lo += (int)row_least_from(key, lo);      // the border is a key: the smallest taken one
    unsigned taken = 0;
#pragma unroll
    for (int j = VPL - 1; j >= 0; --j) taken = taken + taken + (unsigned)(key[j] >= lo);      // lo is above kShut, INT_MAX without open keys
    const int have = row_sum(__popc(taken));
    if (have != n) fine = false;                 // equal keys at the border
    if (direct && a.ngroups > 1 && have > 0) {
        // the values p in 64 bits are in the scores' order unless they saturate or two scores nearly meet at the border
        const float t = key_score<T>(lo);
        if (!(a.kind == 0 ? t - top > -700.f : t > -700.f && t < 20.f)) fine = false;
        if (row_count(key, score_key<T>(t - 0x1p-20f)) != row_count(key, score_key<T>(t))) fine = false;
    }
    if (!direct) {
        // no other key within the errors of two keys below the smallest taken one
        const float t = __int_as_float(lo), e = 2.f * fminf(most, 0x1p-15f * t);
        if (row_count(key, max(kShut + 1, __float_as_int(t - e))) != have) fine = false;
    }
    return taken;
}

template <class T, int VPL, int BLOCK, bool ONE>
__global__ __launch_bounds__(BLOCK) void k_route_rows(RouteArgs a, Deal d, Deal d64, int* shares) {
    constexpr int WAVES = BLOCK / 64;
    __shared__ int hist[16 * VPL < 256 ? 256 : 16 * VPL];
    __shared__ Chosen chosen[WAVES];
    __shared__ int two_largest[WAVES][4][16];
    extern __shared__ double exact_keys[];      // 64 * d64.each per wave
    if (a.counts != nullptr) {
        for (int e = threadIdx.x; e < a.nexperts; e += BLOCK) hist[e] = 0;
        __syncthreads();
    }
    const int l = threadIdx.x & 63, wave = wave_uniform(threadIdx.x >> 6);
    Chosen& ch = chosen[wave];
    const int row = l >> 4, i = l & 15;
    const int g = i / d.lanes, o = (i & (d.lanes - 1)) * d.each;
    const int first = g * d.size + o;
    const int room = d.size - o < d.each ? d.size - o : d.each;
    const int own = g < a.ngroups && room > 0 ? room : 0;
    float bias[VPL];
    int most_bias = 0;          // a NaN stands above infinity here
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
        bias[j] = a.bias != nullptr && j < own ? a.bias[first + j] : 0.f;
        most_bias = max(most_bias, __float_as_int(bias[j]) & 0x7fffffff);
    }
    const float bmax = __int_as_float(wave_max(most_bias));
    const bool exact_only = !(bmax < 0x1p100f);          // the error bounds below are for finite biases
#pragma unroll
    for (int j = 0; j < VPL; ++j) bias[j] += bmax;
    const bool sums = a.kind == 0 && (a.bias != nullptr || a.ngroups > 1 || !a.renorm);
    const bool full = __ballot(own != VPL) == 0;      // every lane has VPL experts
    const long long end = (a.ncols - 1LL) * a.ldz + a.nexperts;
    const long long step = (long long)gridDim.x * WAVES * d.batch;
    for (long long c0 = ((long long)blockIdx.x * WAVES + wave) * d.batch; c0 < a.ncols; c0 += step) {
        const int cols = (int)(a.ncols - c0 < d.batch ? a.ncols - c0 : d.batch);
        for (int b0 = 0; b0 < cols; b0 += 4) {
            const int b = b0 + row;
            const long long c = c0 + (b < cols ? b : cols - 1);      // rows past the end repeat the last column
            const long long at = c * a.ldz + first;
            float z[VPL];
            if (VPL >= 2 && full) {
                T raw[VPL];
                __builtin_memcpy(raw, (const T*)a.Z + at, sizeof(raw));
#pragma unroll
                for (int j = 0; j < VPL; ++j) z[j] = (float)raw[j];
            } else if (VPL >= 2 && at + VPL <= end) {          // wide loads may run into the next column, not out of the matrix
                T raw[VPL];
                __builtin_memcpy(raw, (const T*)a.Z + at, sizeof(raw));
#pragma unroll
                for (int j = 0; j < VPL; ++j) z[j] = j < own ? (float)raw[j] : -INFINITY;
            } else {
#pragma unroll
                for (int j = 0; j < VPL; ++j) z[j] = j < own ? (float)((const T*)a.Z)[at + j] : -INFINITY;
            }
            // a NaN anywhere, or +inf where the softmax has no value
            unsigned size = 0;
#pragma unroll
            for (int j = 0; j < VPL; ++j) size = max(size, (unsigned)__float_as_int(z[j]) & 0x7fffffffu);
            const bool shut = __ballot(size >= 0x7f800000u) != 0;          // some infinity: of -inf, where all is well
            bool odd = size > 0x7f800000u;
            if (shut && a.kind == 0) {
#pragma unroll
                for (int j = 0; j < VPL; ++j) odd = odd || z[j] == INFINITY;
            }
            const bool bad = shut && row_sum(odd) != 0;
            float top = 0.f, by = 1.f;
            if (sums) {
                top = z[0];
#pragma unroll
                for (int j = 1; j < VPL; ++j) top = fmaxf(top, z[j]);
                top = group_allmax<16>(top);
                const float from = top > -INFINITY ? top : 0.f;
                float sum = 0.f;
#pragma unroll
                for (int j = 0; j < VPL; ++j) sum += __builtin_amdgcn_exp2f((z[j] - from) * kLog2e);
                sum = group_allsum<16>(sum);
                by = sum > 0.f ? 1.f / sum : 0.f;
            }
            bool fine;
            unsigned taken = take_row<T, VPL>(a, d, z, bias, bmax, top, by, first, shut, two_largest[wave][row], fine);
            fine = fine && !exact_only;
            if (bad) { taken = 0; fine = true; }
            // fewer than topk open: the lowest others fill the column
            const unsigned valid = taken;
            int upto = row_prefix(__popc(taken));
            const int have = row_sum(__popc(taken));
            if (__ballot(have < a.topk) != 0) {
                unsigned rest = own > 0 ? ~taken & (own >= 32 ? ~0u : (1u << own) - 1u) : 0u;
                int left = a.topk - have - (row_prefix(__popc(rest)) - __popc(rest));
                for (; rest != 0 && left > 0; rest &= rest - 1, --left) taken |= rest & -rest;
                upto = row_prefix(__popc(taken));
            }
            int before = upto - __popc(taken);
            const unsigned long long unclear = __ballot(!fine);
            if (b < cols && (unclear >> (16 * row) & 0xffff) == 0) {
                for (unsigned t = taken; t != 0; t &= t - 1) {
                    const int j = __builtin_ctz(t);
                    ch.row[b][before++] = (unsigned short)((first + j) | (valid >> j & 1 ? 0 : 0x8000));
                }
            }
            if (b < cols && i == 0) {
                ch.top[b] = bad ? NAN : top;
                ch.by[b] = by;
            }
            for (int r = 0; r < 4 && b0 + r < cols; ++r)
                if (unclear >> (16 * r) & 0xffff) exact_column<T>(a, d64, c0 + b0 + r, exact_keys + wave * 64 * d64.each, ch.row[b0 + r]);
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        write_weights<T>(a, d, ch, c0, cols, hist);
        __builtin_amdgcn_wave_barrier();
    }
    if (a.counts != nullptr) {
        __syncthreads();
        for (int e = threadIdx.x; e < a.nexperts; e += BLOCK) {
            if (ONE) a.counts[e] = hist[e];
            else shares[(size_t)blockIdx.x * a.nexperts + e] = hist[e];
        }
    }
}

// Gradient. With w the weights (0: the entry was not taken), dg their gradient and mean = sum of w * dg over the column:
//   softmax                  dz_i = p_i * (scale * dg_i [taken] - mean)
//   softmax, renormalised    dz_i = w_i * (dg_i - mean / scale)                taken entries, 0 elsewhere
//   sigmoid                  dz_i = w_i * (1 - p_i) * dg_i                     likewise
//   sigmoid, renormalised    dz_i = w_i * (1 - p_i) * (dg_i - mean / scale)    likewise
// LPC lanes share a column, eight experts to a lane and turn. The entries' values meet the experts in LDS, so that the
// column is written once.
// What bounds it: memory in large calls (256 experts, 32768 columns in fp32, softmax: 14.8 us, 4.7 TB/s), before that the way
// from a column's rows to its values, which more columns per wave hide: two turns of half the lanes are kept (512
// experts, 32768 columns in bf16: 14.9 us, renormalised 9.6; one turn of 64 lanes 17.8 and 13.9; 128 experts 7.7).
template <class T, int LPC, int NV>
__global__ __launch_bounds__(BM_BLOCK) void k_route_grad(RouteGradArgs a) {
    constexpr int CPW = 64 / LPC;
    __shared__ float at_expert[BM_BLOCK / LPC][LPC * NV * 8];
    const int lane = threadIdx.x & 63, t = lane & (LPC - 1);
    const long long c = ((long long)blockIdx.x * BM_WAVES_PER_BLOCK + (threadIdx.x >> 6)) * CPW + lane / LPC;
    if (c >= a.ncols) return;
    float* up = at_expert[threadIdx.x / LPC];
    const T* z = (const T*)a.Z + c * a.ldz;
    const int n = a.nexperts;
    const bool dense = a.kind == 0 && !a.renorm;
    const long long q0 = c * a.topk;
    float mean = 0.f;
    for (int s = t; s < a.topk; s += LPC) {
        const float w = (unsigned)a.ir[q0 + s] < (unsigned)n ? a.data[q0 + s] : 0.f;
        if (w != 0.f) mean += w * a.ddata[q0 + s];
    }
    mean = group_allsum<LPC>(mean);
    float8_t x[NV];
    float by = 0.f, top = -INFINITY;
    if (dense) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            x[v] = load_col8(z, (v * LPC + t) * 8, n, (T)(-INFINITY)).wide();
#pragma unroll
            for (int j = 0; j < 8; ++j) top = fmaxf(top, x[v][j]);
        }
        top = group_allmax<LPC>(top);
        if (top == -INFINITY) top = 0.f;
        float sum = 0.f;
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[v][j] = __builtin_amdgcn_exp2f((x[v][j] - top) * kLog2e);
                sum += x[v][j];
            }
        sum = group_allsum<LPC>(sum);
        by = sum == 0.f ? 0.f : 1.f / sum;              // a column without open experts; a NaN stays one
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) *(float8_t*)(up + (v * LPC + t) * 8) = (float8_t)(0.f);
    __builtin_amdgcn_wave_barrier();                    // a wave's LDS operations take effect in order
    for (int s = t; s < a.topk; s += LPC) {
        const int r = a.ir[q0 + s];
        if ((unsigned)r >= (unsigned)n) continue;
        const float w = a.data[q0 + s], dg = a.ddata[q0 + s];
        if (w == 0.f) continue;
        float d = dense ? a.scale * dg : w * (a.renorm ? dg - mean / a.scale : dg);
        if (a.kind == 1) d *= 1.f / (1.f + expf((float)z[r]));
        if (w != w) d = w;
        up[r] = d;
    }
    __builtin_amdgcn_wave_barrier();
    T* dz = (T*)a.dZ + c * a.lddz;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        float8_t d = *(const float8_t*)(up + (v * LPC + t) * 8);
        if (dense) d = x[v] * by * (d - mean);
        store_col8(dz, (v * LPC + t) * 8, n, d);
    }
}

// counts[e] = sum of the workgroups' shares (atomics of a thousand workgroups on one address took longer than the rest): 16
// experts x 64 threads.
__global__ __launch_bounds__(1024) void k_add_counts(int n, int nshares, const int* __restrict__ shares, int* __restrict__ counts) {
    __shared__ int sh[64][17];
    const int x = threadIdx.x & 15, y = threadIdx.x >> 4, e = blockIdx.x * 16 + x;
    int c = 0;
    if (e < n)
#pragma unroll 8
        for (int p = y; p < nshares; p += 64) c += shares[(size_t)p * n + e];
    sh[y][x] = c;
    for (int step = 32; step > 0; step >>= 1) {
        __syncthreads();
        if (y < step) sh[y][x] += sh[y + step][x];
    }
    if (y == 0 && e < n) counts[e] = sh[0][x];
}
hipError_t count_shares(const RouteArgs& a, unsigned grid, int** shares, hipStream_t s) {
    hipError_t e = hipSuccess;
    *shares = nullptr;
    if (a.counts != nullptr) *shares = (int*)ws_get(WS_ROUTE, sizeof(int) * (size_t)grid * a.nexperts, &e, s);
    return e;
}
hipError_t add_counts(const RouteArgs& a, unsigned grid, const int* shares, hipStream_t s) {
    if (a.counts != nullptr)
        hipLaunchKernelGGL(k_add_counts, dim3((a.nexperts + 15) / 16), dim3(1024), 0, s, a.nexperts, (int)grid, shares, a.counts);
    return hipGetLastError();
}

// Few columns are left to one workgroup, which writes the counts itself and saves the second launch (7.4 us a call instead of
// 9.8): up to two columns per wave (384 experts: 16 columns 10.7 us, 32 17.2 us against 10.9 by many workgroups), or, with
// 16 lanes to a column, kOneRows (128 experts: 32 columns 7.3 us, by one column per wave 9.3; 64 columns 9.1; 256 experts: 48
// columns 8.4 us against 9.8 by many workgroups, but in 8 groups, for which there is no border of its own, 13.2 against 10.7).
constexpr int kOneRows = 48, kOneColumns = 2;
// Waves per workgroup: as many as leave the keys of take_exact 32 KiB of LDS.
constexpr int route_waves(int vpl, bool one) { return vpl <= 4 ? (one ? 16 : 8) : 64 / vpl; }

template <class T, int VPL>
hipError_t launch_route(const RouteArgs& a, Deal d, hipStream_t s) {
    const size_t keys = 64 * sizeof(double) * d.each;      // of one wave
    if (a.ncols <= kOneColumns * route_waves(VPL, true)) {
        constexpr int waves = route_waves(VPL, true);
        d.batch = (a.ncols + waves - 1) / waves < kRouteBatch ? (a.ncols + waves - 1) / waves : kRouteBatch;
        hipLaunchKernelGGL((k_route<T, VPL, 64 * waves, true>), dim3(1), dim3(64 * waves), waves * keys, s, a, d, (int*)nullptr);
        return hipGetLastError();
    }
    constexpr int waves = route_waves(VPL, false);
    const long long all = 16384;      // waves that keep the device busy: fewer columns per wave rather than fewer waves
    d.batch = a.ncols >= all * kRouteBatch ? kRouteBatch : (int)((a.ncols + all - 1) / all);
    const long long want = (a.ncols + (long long)waves * d.batch - 1) / (waves * d.batch), most = 8192 / waves;
    const unsigned grid = (unsigned)(want < most ? want : most);
    int* shares;
    const hipError_t e = count_shares(a, grid, &shares, s);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((k_route<T, VPL, 64 * waves, false>), dim3(grid), dim3(64 * waves), waves * keys, s, a, d, shares);
    return add_counts(a, grid, shares, s);
}

template <class T, int VPL>
hipError_t launch_route_rows(const RouteArgs& a, Deal d, const Deal& d64, hipStream_t s) {
    const size_t keys = 64 * sizeof(double) * d64.each;      // of one wave
    if constexpr (VPL <= 16) if (a.ncols <= kOneRows) {
        d.batch = 4;
        hipLaunchKernelGGL((k_route_rows<T, VPL, 1024, true>), dim3(1), dim3(1024), 16 * keys, s, a, d, d64, (int*)nullptr);
        return hipGetLastError();
    }
    const long long all = 4096;
    d.batch = a.ncols >= all * 4 ? 8 : 4;
    const long long want = (a.ncols + BM_WAVES_PER_BLOCK * (long long)d.batch - 1) / (BM_WAVES_PER_BLOCK * d.batch);
    const unsigned grid = (unsigned)(want < all / BM_WAVES_PER_BLOCK ? want : all / BM_WAVES_PER_BLOCK);
    int* shares;
    const hipError_t e = count_shares(a, grid, &shares, s);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((k_route_rows<T, VPL, BM_BLOCK, false>), dim3(grid), dim3(BM_BLOCK), BM_WAVES_PER_BLOCK * keys, s, a, d, d64, shares);
    return add_counts(a, grid, shares, s);
}

Deal deal(const RouteArgs& a, int lanes) {
    Deal d;
    d.size = a.nexperts / a.ngroups;
    d.lanes = lanes / pow2ceil(a.ngroups);
    d.each = d.lanes > 0 ? (d.size + d.lanes - 1) / d.lanes : INT_MAX;
    d.kp = pow2ceil(a.topk);
    d.batch = 1;
    d.halves = a.topgroups * d.lanes <= 8;
    return d;
}

template <class T>
hipError_t route_typed(const RouteArgs& a, hipStream_t s) {
    const Deal d = deal(a, 64), d16 = deal(a, 16);
    // four columns per wave, once a workgroup's sixteen waves have a column each (with up to 32 experts in a lane, four times as
    // many: 512 experts, 17 columns 15.7 us, by a wave per column 12.2, 100 columns 15.5 and 16.6, 32768 columns bf16 48 and 70)
    if (a.ncols > (d16.each <= 16 ? 16 : 64) && d16.each <= 32 && a.nexperts <= 512 && a.topk <= 16) {
        if (d16.each <= 1) return launch_route_rows<T, 1>(a, d16, d, s);
        if (d16.each <= 2) return launch_route_rows<T, 2>(a, d16, d, s);
        if (d16.each <= 4) return launch_route_rows<T, 4>(a, d16, d, s);
        if (d16.each <= 8) return launch_route_rows<T, 8>(a, d16, d, s);
        if (d16.each <= 16) return launch_route_rows<T, 16>(a, d16, d, s);
        return launch_route_rows<T, 32>(a, d16, d, s);
    }
    if (d.each <= 1) return launch_route<T, 1>(a, d, s);
    if (d.each <= 2) return launch_route<T, 2>(a, d, s);
    if (d.each <= 4) return launch_route<T, 4>(a, d, s);
    if (d.each <= 8) return launch_route<T, 8>(a, d, s);
    if (d.each <= 16) return launch_route<T, 16>(a, d, s);
    return launch_route<T, 32>(a, d, s);
}

}  // namespace

hipError_t route(const RouteArgs& a, hipStream_t s) {
    return a.type == ELEM_F32 ? route_typed<float>(a, s) : a.type == ELEM_F16 ? route_typed<f16_t>(a, s) : route_typed<bf16_t>(a, s);
}

namespace {
template <class T, int LPC, int NV>
hipError_t launch_route_grad(const RouteGradArgs& a, hipStream_t s) {
    constexpr int CPB = BM_BLOCK / LPC;
    hipLaunchKernelGGL((k_route_grad<T, LPC, NV>), dim3((unsigned)((a.ncols + CPB - 1LL) / CPB)), dim3(BM_BLOCK), 0, s, a);
    return hipGetLastError();
}
template <class T>
hipError_t route_grad_typed(const RouteGradArgs& a, hipStream_t s) {
    if (a.nexperts <= 64) return launch_route_grad<T, 8, 1>(a, s);
    if (a.nexperts <= 128) return launch_route_grad<T, 8, 2>(a, s);
    if (a.nexperts <= 256) return launch_route_grad<T, 16, 2>(a, s);
    if (a.nexperts <= 512) return launch_route_grad<T, 32, 2>(a, s);
    return launch_route_grad<T, 64, 2>(a, s);
}
}  // namespace

hipError_t route_grad(const RouteGradArgs& all, hipStream_t s) {
    const long long size = (long long)elem_size(all.type);
    for (long long c = 0; c < all.ncols; c += kSlabColumns) {
        RouteGradArgs a = all;
        a.ncols = (int)(all.ncols - c < kSlabColumns ? all.ncols - c : kSlabColumns);
        a.Z = (const char*)all.Z + c * all.ldz * size;
        a.dZ = (char*)all.dZ + c * all.lddz * size;
        a.data = all.data + c * all.topk;
        a.ir = all.ir + c * all.topk;
        a.ddata = all.ddata + c * all.topk;
        const hipError_t e = a.type == ELEM_F32 ? route_grad_typed<float>(a, s) : a.type == ELEM_F16 ? route_grad_typed<f16_t>(a, s) : route_grad_typed<bf16_t>(a, s);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace bm
