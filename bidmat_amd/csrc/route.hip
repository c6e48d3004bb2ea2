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
#include "columns.hpp"
#include "elems.hpp"
#include "kernels.hpp"

namespace bm {
namespace {

constexpr float kLog2e = 1.44269504088896340736f;

struct Deal {            // how a column's experts lie in the lanes
    int lanes;           // lanes per group (a power of two)
    int size;            // experts per group
    int each;            // experts per lane
    int kp;              // topk rounded up to a power of two: lanes per column when the weights are written
    int batch;           // columns whose weights a wave writes together
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
// Largest value of the wave in a scalar register: shifts inside rows of 16 lanes, then row results broadcast onwards.
__device__ __forceinline__ float wave_max(float x) {
    constexpr int low = (int)0xff800000;      // -inf
#define BM_STEP(ctrl, rows) x = fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp(low, __float_as_int(x), ctrl, rows, 0xf, false)))
    BM_STEP(0x111, 0xf); BM_STEP(0x112, 0xf); BM_STEP(0x114, 0xf); BM_STEP(0x118, 0xf);      // row_shr 1, 2, 4, 8
    BM_STEP(0x142, 0xa); BM_STEP(0x143, 0xc);                                                // row_bcast 15, 31
#undef BM_STEP
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}
__device__ __forceinline__ float wave_sum(float x) {
#define BM_STEP(ctrl, rows) x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), ctrl, rows, 0xf, false))
    BM_STEP(0x111, 0xf); BM_STEP(0x112, 0xf); BM_STEP(0x114, 0xf); BM_STEP(0x118, 0xf);
    BM_STEP(0x142, 0xa); BM_STEP(0x143, 0xc);
#undef BM_STEP
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}

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
__device__ __forceinline__ int count_from(const float (&key)[N], float t) {
    int c = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) c += __popcll(__ballot(key[j] >= t));
    return c;
}

// The border below the `want` largest of the wave's keys (more than want are above -inf): they are the keys >= t, of
// those that equal t only the first `ties` when ties > 0. `between`: t is no key but lies between two.
struct Border { float t; int ties; bool between; };
template <int N>
__device__ __forceinline__ Border find_border(const float (&key)[N], int want) {
    float best = key[0];
#pragma unroll
    for (int j = 1; j < N; ++j) best = fmaxf(best, key[j]);
    const float top = wave_max(best);
    // every lane's largest key but those of lanes without an open one: at least as many keys reach the least of them
    float lo = -wave_max(best > -INFINITY ? -best : -INFINITY);
    int n = count_from(key, lo);
    if (n < want) {
        float least = INFINITY;
#pragma unroll
        for (int j = 0; j < N; ++j) least = fminf(least, key[j] > -INFINITY ? key[j] : INFINITY);
        lo = -wave_max(-least);
        n = count_from(key, lo);
    }
    float hi = NAN;                 // none yet: no comparison with it holds
    int above = 0;
    if (n == want) return {lo, 0, false};
    for (int i = 0; i < 14; ++i) {
        const float end = hi < top ? hi : top, mid = 0.5f * lo + 0.5f * end;
        if (!(mid > lo && mid < end)) break;
        const int c = count_from(key, mid);
        if (c == want) return {mid, 0, true};
        if (c > want) lo = mid; else { hi = mid; above = c; }
    }
    // what is left lies close together: one value at a time from above
    for (;;) {
        float next = -INFINITY;
#pragma unroll
        for (int j = 0; j < N; ++j) next = fmaxf(next, key[j] >= hi ? -INFINITY : key[j]);
        next = wave_max(next);
        int c = 0;
#pragma unroll
        for (int j = 0; j < N; ++j) c += __popcll(__ballot(key[j] == next));
        if (above + c >= want || !(next > -INFINITY)) return {next, above + c > want ? want - above : 0, false};
        above += c;
        hi = next;
    }
}
// Whether keys that are off by at most e each have the same largest `want` as the exact ones.
template <int N>
__device__ __forceinline__ bool border_clear(const float (&key)[N], const Border& b, int want, float e) {
    if (b.ties > 0) return false;
    if (b.between) return count_from(key, b.t + e) == want && count_from(key, b.t - e) == want;
    return count_from(key, b.t - 2.f * e) == want;
}

// The same in fp32; false: some key lies too close to a border.
template <int VPL>
__device__ __forceinline__ bool take_fast(const RouteArgs& a, const Deal& d, const float (&z)[VPL], const float (&bias)[VPL], float bmax,
                                          float top, float by, unsigned& taken) {
    const int l = threadIdx.x & 63;
    const bool plain = a.bias == nullptr && a.ngroups == 1;
    float key[VPL];
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
        if (plain) key[j] = z[j];
        else if (a.kind == 0) key[j] = __builtin_amdgcn_exp2f((z[j] - top) * kLog2e) * by;
        else key[j] = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-z[j] * kLog2e));
        if (!plain) {
            key[j] += bias[j];
            key[j] = z[j] > -INFINITY && key[j] > -INFINITY ? key[j] : -INFINITY;
        }
    }
    // Error of a key near the value v: p = key - bias is off by up to 2^-16 of itself (exp of an argument of up to 88, the
    // sum), a sigmoid also by less than 2^-20 at all.
    const float most = a.kind == 0 ? INFINITY : 0x1p-20f * (1.f + bmax);
    if (a.ngroups > 1) {
        float best = key[0], second = -INFINITY;
#pragma unroll
        for (int j = 1; j < VPL; ++j) {
            second = fmaxf(second, fminf(best, key[j]));
            best = fmaxf(best, key[j]);
        }
        auto merge = [&](float ob, float os) {
            second = fmaxf(fminf(best, ob), fmaxf(second, os));
            best = fmaxf(best, ob);
        };
        if (d.lanes >= 2) merge(dpp_mov<DPP_QUAD_XOR1>(best), dpp_mov<DPP_QUAD_XOR1>(second));
        if (d.lanes >= 4) merge(dpp_mov<DPP_QUAD_XOR2>(best), dpp_mov<DPP_QUAD_XOR2>(second));
        if (d.lanes >= 8) merge(dpp_mov<DPP_ROW_HALF_MIRROR>(best), dpp_mov<DPP_ROW_HALF_MIRROR>(second));
        if (d.lanes >= 16) merge(dpp_mov<DPP_ROW_MIRROR>(best), dpp_mov<DPP_ROW_MIRROR>(second));
        if (d.lanes >= 32) merge(__shfl_xor(best, 16, 64), __shfl_xor(second, 16, 64));
        const float mine = second > -INFINITY ? best + second : best;
        // one lane of each group stands for it
        float score[1] = {(l & (d.lanes - 1)) == 0 ? mine : -INFINITY};
        if (__popcll(__ballot(score[0] > -INFINITY)) > a.topgroups) {
            const Border b = find_border(score, a.topgroups);
            if (!border_clear(score, b, a.topgroups, fminf(2.f * most, 0x1p-15f * (fabsf(b.t) + 2.f * bmax)))) return false;
            if (!(mine >= b.t)) {
#pragma unroll
                for (int j = 0; j < VPL; ++j) key[j] = -INFINITY;
            }
        }
    }
    taken = 0;
    int open = 0;
#pragma unroll
    for (int j = 0; j < VPL; ++j) open += __popcll(__ballot(key[j] > -INFINITY));
    if (open <= a.topk) {
#pragma unroll
        for (int j = 0; j < VPL; ++j) taken |= key[j] > -INFINITY ? 1u << j : 0u;
        return true;
    }
    const Border b = find_border(key, a.topk);
    if (!plain && !border_clear(key, b, a.topk, fminf(most, 0x1p-16f * (fabsf(b.t) + bmax)))) return false;
#pragma unroll
    for (int j = 0; j < VPL; ++j) taken |= key[j] >= b.t ? 1u << j : 0u;
    if (b.ties > 0) {
        // exact keys: of those that equal the border the first ones stay
        unsigned equal = 0;
#pragma unroll
        for (int j = 0; j < VPL; ++j) equal |= key[j] == b.t ? 1u << j : 0u;
        int mine = __popc(equal), before = mine;
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
            const int y = __shfl_up(before, m, 64);
            if (l >= m) before += y;
        }
        int left = b.ties - (before - mine);
#pragma unroll
        for (int j = 0; j < VPL; ++j)
            if (equal >> j & 1) {
                if (left <= 0) taken &= ~(1u << j);
                --left;
            }
    }
    return true;
}

// Sum / largest over aligned groups of n lanes, n a power of two known at run time.
__device__ __forceinline__ float lanes_sum_rt(float x, int n) {
    for (int m = 1; m < n; m <<= 1) x += __shfl_xor(x, m, 64);
    return x;
}
__device__ __forceinline__ float lanes_max_rt(float x, int n) {
    for (int m = 1; m < n; m <<= 1) x = fmaxf(x, __shfl_xor(x, m, 64));
    return x;
}

constexpr int kRouteBatch = 8;           // columns whose weights one wave writes together, at most
struct Chosen {                          // of one wave
    unsigned short row[kRouteBatch][kRouteMaxTop];      // bit 15: named only to fill the column, weight 0
    float top[kRouteBatch], by[kRouteBatch];            // softmax over all: p = exp(z - top) * by; top NaN: the column holds one
};

// BLOCK threads; ONE: a single workgroup, which writes the counts instead of adding to them.
template <class T, int VPL, int BLOCK, bool ONE>
__global__ __launch_bounds__(BLOCK) void k_route(RouteArgs a, Deal d) {
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
    float bias[VPL], bmax = 0.f;
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
        bias[j] = a.bias != nullptr && j < own ? a.bias[first + j] : 0.f;
        bmax = fmaxf(bmax, fabsf(bias[j]));
    }
    bmax = wave_max(bmax);
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
            bool odd = false;
#pragma unroll
            for (int j = 0; j < VPL; ++j) odd = odd || z[j] != z[j] || (a.kind == 0 && z[j] == INFINITY);
            const bool bad = __ballot(odd) != 0;
            float top = 0.f, by = 1.f;
            if (sums) {
                top = z[0];
#pragma unroll
                for (int j = 1; j < VPL; ++j) top = fmaxf(top, z[j]);
                top = wave_max(top);
                float sum = 0.f;
#pragma unroll
                for (int j = 0; j < VPL; ++j) sum += z[j] > -INFINITY ? __builtin_amdgcn_exp2f((z[j] - top) * kLog2e) : 0.f;
                sum = wave_sum(sum);
                by = sum > 0.f ? 1.f / sum : 0.f;
            }
            unsigned taken = 0;
            if (!bad && !take_fast<VPL>(a, d, z, bias, bmax, top, by, taken)) 
                taken = take_exact<T>((const T*)a.Z + at, a.bias != nullptr ? a.bias + first : nullptr, exact_keys + wave * 64 * d.each, own,
                                      d.each, a.kind, a.ngroups, a.topgroups, a.topk, d.lanes);
            // fewer than topk open: the lowest others fill the column
            const unsigned valid = taken;
            const int mine = __popc(taken);
            int before = mine, have;
            {
                // lanes hold at most a few: prefix over the wave
                int s = mine;
#pragma unroll
                for (int m = 1; m < 64; m <<= 1) {
                    const int y = __shfl_up(s, m, 64);
                    if (l >= m) s += y;
                }
                have = __builtin_amdgcn_readlane(s, 63);
                before = s - mine;
            }
            if (have < a.topk) {
                const unsigned rest = own > 0 ? ~taken & (own >= 32 ? ~0u : (1u << own) - 1u) : 0u;
                const int n = __popc(rest);
                int s = n;
#pragma unroll
                for (int m = 1; m < 64; m <<= 1) {
                    const int y = __shfl_up(s, m, 64);
                    if (l >= m) s += y;
                }
                int left = a.topk - have - (s - n);
#pragma unroll
                for (int j = 0; j < VPL; ++j)
                    if ((rest >> j & 1) && left > 0) { taken |= 1u << j; --left; }
                s = __popc(taken);
#pragma unroll
                for (int m = 1; m < 64; m <<= 1) {
                    const int y = __shfl_up(s, m, 64);
                    if (l >= m) s += y;
                }
                before = s - __popc(taken);
            }
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
        // the weights: kp lanes per column
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
                p = a.kind == 0 || high < -30.f ? expf(z - high) : 1.f / (1.f + expf(-z));
                p = valid ? p : 0.f;
                const float sum = lanes_sum_rt(p, d.kp);
                p = sum > 0.f ? p * (a.scale / sum) : 0.f;
            } else {
                p = a.scale * (a.kind == 0 ? expf(z - top) * by : 1.f / (1.f + expf(-z)));
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
        __builtin_amdgcn_wave_barrier();
    }
    if (a.counts != nullptr) {
        // whole numbers: the same total in any order
        __syncthreads();
        for (int e = threadIdx.x; e < a.nexperts; e += BLOCK) {
            if (ONE) a.counts[e] = hist[e];
            else if (hist[e] != 0) atomicAdd(&a.counts[e], hist[e]);
        }
    }
}

// Gradient. With w the weights (0: the entry was not taken), dg their gradient and mean = sum of w * dg over the column:
//   softmax                  dz_i = p_i * (scale * dg_i [taken] - mean)
//   softmax, renormalised    dz_i = w_i * (dg_i - mean / scale)                taken entries, 0 elsewhere
//   sigmoid                  dz_i = w_i * (1 - p_i) * dg_i                     likewise
//   sigmoid, renormalised    dz_i = w_i * (1 - p_i) * (dg_i - mean / scale)    likewise
// One wave per column: it writes the column (the softmax form from its scores), then its own entries over it.
template <class T>
__global__ __launch_bounds__(BM_BLOCK) void k_route_grad(RouteGradArgs a) {
    const int lane = threadIdx.x & 63;
    const long long c = (long long)blockIdx.x * BM_WAVES_PER_BLOCK + (threadIdx.x >> 6);
    if (c >= a.ncols) return;
    const T* z = (const T*)a.Z + c * a.ldz;
    T* dz = (T*)a.dZ + c * a.lddz;
    const bool mine = lane < a.topk;
    const long long q = c * a.topk + lane;
    const int r = mine ? a.ir[q] : -1;
    const bool ok = mine && (unsigned)r < (unsigned)a.nexperts;
    const float w = ok ? a.data[q] : 0.f, dg = ok ? a.ddata[q] : 0.f;
    const float mean = group_allsum<64>(w == 0.f ? 0.f : w * dg);
    const bool dense = a.kind == 0 && !a.renorm;
    float top = -INFINITY, sum = 0.f, zr = 0.f;
    if (ok && (dense || a.kind == 1)) zr = (float)z[r];
    if (dense) {
        for (int i = lane; i < a.nexperts; i += 64) top = fmaxf(top, (float)z[i]);
        top = group_allmax<64>(top);
        if (top == -INFINITY) top = 0.f;
        for (int i = lane; i < a.nexperts; i += 64) sum += expf((float)z[i] - top);
        sum = group_allsum<64>(sum);
    }
    const float by = sum == 0.f ? 0.f : 1.f / sum;      // a column without open experts; a NaN stays one
    for (int i = lane; i < a.nexperts; i += 64) dz[i] = (T)(dense ? -(expf((float)z[i] - top) * by) * mean : 0.f);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
    if (ok) {
        float d = 0.f;
        if (w != 0.f) {
            if (dense) d = expf(zr - top) * by * (a.scale * dg - mean);
            else d = w * (a.renorm ? dg - mean / a.scale : dg) * (a.kind == 1 ? 1.f / (1.f + expf(zr)) : 1.f);
        } else if (dense) {
            d = -(expf(zr - top) * by) * mean;
        }
        dz[r] = (T)d;
    }
}

constexpr int kOneColumns = 64;          // up to so many columns one workgroup does it all, in one launch
// Waves per workgroup: as many as leave the keys of take_exact 32 KiB of LDS.
constexpr int route_waves(int vpl, bool one) { return vpl <= 4 ? (one ? 16 : 8) : 64 / vpl; }

template <class T, int VPL>
hipError_t launch_route(const RouteArgs& a, Deal d, hipStream_t s) {
    const size_t keys = 64 * sizeof(double) * d.each;      // of one wave
    if (a.ncols <= kOneColumns) {
        constexpr int waves = route_waves(VPL, true);
        d.batch = (a.ncols + waves - 1) / waves < kRouteBatch ? (a.ncols + waves - 1) / waves : kRouteBatch;
        hipLaunchKernelGGL((k_route<T, VPL, 64 * waves, true>), dim3(1), dim3(64 * waves), waves * keys, s, a, d);
        return hipGetLastError();
    }
    if (a.counts != nullptr) {
        const hipError_t e = fill_i32(a.counts, a.nexperts, 0, s);
        if (e != hipSuccess) return e;
    }
    constexpr int waves = route_waves(VPL, false);
    const long long all = 16384;      // waves that keep the device busy: fewer columns per wave rather than fewer waves
    d.batch = a.ncols >= all * kRouteBatch ? kRouteBatch : (int)((a.ncols + all - 1) / all);
    const long long want = (a.ncols + (long long)waves * d.batch - 1) / (waves * d.batch), most = 8192 / waves;
    const unsigned grid = (unsigned)(want < most ? want : most);
    hipLaunchKernelGGL((k_route<T, VPL, 64 * waves, false>), dim3(grid), dim3(64 * waves), waves * keys, s, a, d);
    return hipGetLastError();
}

template <class T>
hipError_t route_typed(const RouteArgs& a, hipStream_t s) {
    Deal d;
    d.size = a.nexperts / a.ngroups;
    d.lanes = 64 / pow2ceil(a.ngroups);
    d.each = (d.size + d.lanes - 1) / d.lanes;
    d.kp = pow2ceil(a.topk);
    d.batch = 1;
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

hipError_t route_grad(const RouteGradArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)((a.ncols + BM_WAVES_PER_BLOCK - 1LL) / BM_WAVES_PER_BLOCK)), block(BM_BLOCK);
    if (a.type == ELEM_F32) hipLaunchKernelGGL((k_route_grad<float>), grid, block, 0, s, a);
    else if (a.type == ELEM_F16) hipLaunchKernelGGL((k_route_grad<f16_t>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((k_route_grad<bf16_t>), grid, block, 0, s, a);
    return hipGetLastError();
}

}  // namespace bm
