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
// LPC lanes of a wave share a column. The groups are dealt to lanes in order, a power of two of lanes to each, and a
// lane holds consecutive experts, so that the order of (lane, slot) is the order of the experts.
#include "columns.hpp"
#include "elems.hpp"
#include "kernels.hpp"

namespace bm {
namespace {

struct Deal {            // how a column's experts lie in its lanes
    int lanes;           // lanes per group (a power of two)
    int size;            // experts per group
    int each;            // experts per lane
};

template <int LPC, class V>
__device__ __forceinline__ V lanes_max(V x) {
#pragma unroll
    for (int m = 1; m < LPC; m <<= 1) {
        const V y = __shfl_xor(x, m, LPC);
        x = y > x ? y : x;
    }
    return x;
}
template <int LPC, class V>
__device__ __forceinline__ V lanes_min(V x) {
#pragma unroll
    for (int m = 1; m < LPC; m <<= 1) {
        const V y = __shfl_xor(x, m, LPC);
        x = y < x ? y : x;
    }
    return x;
}
template <int LPC, class V>
__device__ __forceinline__ V lanes_sum(V x) {
#pragma unroll
    for (int m = 1; m < LPC; m <<= 1) x += __shfl_xor(x, m, LPC);
    return x;
}
// Sum over the lanes before this one.
template <int LPC>
__device__ __forceinline__ int lanes_before(int x) {
    const int l = threadIdx.x & (LPC - 1);
    int s = x;
#pragma unroll
    for (int m = 1; m < LPC; m <<= 1) {
        const int y = __shfl_up(s, m, LPC);
        if (l >= m) s += y;
    }
    return s - x;
}

// Which of a column's experts are taken, from keys in 64 bits: bit j of the result is this lane's slot j.
template <int LPC, int VPL>
__device__ unsigned take_exact(const RouteArgs& a, const Deal& d, const float (&z)[VPL], const float* bias, int l, int first, int own) {
    const double ninf = -__builtin_inf();
    double key[VPL];
    const bool plain = a.bias == nullptr && a.ngroups == 1;
    if (a.kind == 0 && !plain) {
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < VPL; ++j) top = fmaxf(top, z[j]);
        top = lanes_max<LPC>(top);
        double sum = 0.;
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
            key[j] = z[j] > -INFINITY ? exp((double)z[j] - (double)top) : 0.;
            sum += key[j];
        }
        sum = lanes_sum<LPC>(sum);
#pragma unroll
        for (int j = 0; j < VPL; ++j) key[j] /= sum;
    } else {
#pragma unroll
        for (int j = 0; j < VPL; ++j) key[j] = plain ? (double)z[j] : 1. / (1. + exp(-(double)z[j]));
    }
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
        if (a.bias != nullptr && j < own) key[j] += (double)bias[first + j];
        if (!(z[j] > -INFINITY) || !(key[j] > ninf)) key[j] = ninf;
    }
    if (a.ngroups > 1) {
        double best = ninf, second = ninf;
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
            const double low = key[j] < best ? key[j] : best;
            second = low > second ? low : second;
            best = key[j] > best ? key[j] : best;
        }
        for (int m = 1; m < d.lanes; m <<= 1) {
            const double ob = __shfl_xor(best, m, LPC), os = __shfl_xor(second, m, LPC);
            const double low = ob < best ? ob : best, high = os > second ? os : second;
            second = low > high ? low : high;
            best = ob > best ? ob : best;
        }
        const double mine = second > ninf ? best + second : best;
        const int g = l / d.lanes;
        int before = 0;
        for (int q = 0; q < a.ngroups; ++q) {
            const double other = __shfl(mine, q * d.lanes, LPC);
            before += other > mine || (other == mine && q < g);
        }
        if (before >= a.topgroups) {
#pragma unroll
            for (int j = 0; j < VPL; ++j) key[j] = ninf;
        }
    }
    unsigned taken = 0;
    for (int r = 0; r < a.topk; ++r) {
        double best = ninf;
        int at = 0;
#pragma unroll
        for (int j = 0; j < VPL; ++j)
            if (!(taken >> j & 1) && key[j] > best) { best = key[j]; at = j; }
        const double top = lanes_max<LPC>(best);
        if (!(top > ninf)) break;
        const int who = lanes_min<LPC>(best == top ? l : LPC);
        if (who == l) taken |= 1u << at;
    }
    return taken;
}

template <class T, int LPC, int VPL>
__global__ __launch_bounds__(BM_BLOCK) void k_route(RouteArgs a, Deal d) {
    constexpr int CPB = BM_BLOCK / LPC;
    __shared__ int hist[kRouteMaxExperts];
    if (a.counts != nullptr) {
        for (int e = threadIdx.x; e < a.nexperts; e += BM_BLOCK) hist[e] = 0;
        __syncthreads();
    }
    const int l = threadIdx.x & (LPC - 1);
    const int g = l / d.lanes, o = (l & (d.lanes - 1)) * d.each;       // group of this lane, first slot inside it
    const int first = g * d.size + o;
    const int own = g < a.ngroups ? (d.size - o < d.each ? d.size - o : d.each) : 0;      // may be below 0: none
    for (long long c = (long long)blockIdx.x * CPB + threadIdx.x / LPC; c < a.ncols; c += (long long)gridDim.x * CPB) {
        const T* zp = (const T*)a.Z + c * a.ldz + first;
        float z[VPL];
        bool bad = false;
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
            z[j] = j < own ? (float)zp[j] : -INFINITY;
            bad = bad || z[j] != z[j] || (a.kind == 0 && z[j] == INFINITY);
        }
        bad = lanes_max<LPC>((int)bad) != 0;
        unsigned taken = bad ? 0u : take_exact<LPC, VPL>(a, d, z, a.bias, l, first, own);
        const unsigned valid = taken;
        // fewer than topk are open: the lowest others, with weight 0
        const int have = lanes_sum<LPC>(__popc(taken));
        if (have < a.topk) {
            const unsigned rest = own > 0 ? ~taken & (own >= 32 ? ~0u : (1u << own) - 1u) : 0u;
            int left = a.topk - have - lanes_before<LPC>(__popc(rest));
#pragma unroll
            for (int j = 0; j < VPL; ++j)
                if ((rest >> j & 1) && left > 0) { taken |= 1u << j; --left; }
        }
        // the weights
        float p[VPL], sum = 0.f;
        float top = -INFINITY;
        if (a.kind == 0 || a.renorm) {
#pragma unroll
            for (int j = 0; j < VPL; ++j)
                if (!a.renorm || (valid >> j & 1)) top = fmaxf(top, z[j]);
            top = lanes_max<LPC>(top);
        }
        // Far below 0 sigmoid(z) is exp(z) to within a factor 1 + exp(z): with all taken scores below -30 their
        // shares are a softmax's, where the sigmoids themselves may have left the range of fp32.
        const bool soft = a.kind == 0 || (a.renorm && top < -30.f);
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
            p[j] = soft ? expf(z[j] - top) : 1.f / (1.f + expf(-z[j]));
            if (a.kind == 0 && !a.renorm ? z[j] > -INFINITY : (valid >> j & 1) != 0) sum += p[j];
        }
        sum = lanes_sum<LPC>(sum);
        const float by = a.kind == 0 || a.renorm ? (sum > 0.f ? a.scale / sum : 0.f) : a.scale;
        int at = lanes_before<LPC>(__popc(taken));
#pragma unroll
        for (int j = 0; j < VPL; ++j)
            if (taken >> j & 1) {
                const long long q = c * a.topk + at++;
                a.ir[q] = first + j;
                a.data[q] = bad ? NAN : (valid >> j & 1) ? p[j] * by : 0.f;
                if (a.ic != nullptr) a.ic[q] = (int)c;
                if (a.counts != nullptr && (valid >> j & 1)) atomicAdd(&hist[first + j], 1);
            }
        if (l == 0 && a.jc != nullptr) {
            a.jc[c] = (int)(c * a.topk);
            if (c == a.ncols - 1) a.jc[c + 1] = (int)((c + 1) * a.topk);
        }
    }
    if (a.counts != nullptr) {
        // whole numbers: the same total in any order
        __syncthreads();
        for (int e = threadIdx.x; e < a.nexperts; e += BM_BLOCK)
            if (hist[e] != 0) atomicAdd(&a.counts[e], hist[e]);
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

template <class T, int LPC, int VPL>
hipError_t launch_route(const RouteArgs& a, const Deal& d, hipStream_t s) {
    constexpr int CPB = BM_BLOCK / LPC;
    const long long want = (a.ncols + CPB - 1LL) / CPB;
    const unsigned grid = (unsigned)(want < 1024 ? want : 1024);
    hipLaunchKernelGGL((k_route<T, LPC, VPL>), dim3(grid), dim3(BM_BLOCK), 0, s, a, d);
    return hipGetLastError();
}

template <class T>
hipError_t route_typed(const RouteArgs& a, hipStream_t s) {
    Deal d;
    d.size = a.nexperts / a.ngroups;
    d.lanes = 64 / pow2ceil(a.ngroups);
    d.each = (d.size + d.lanes - 1) / d.lanes;
    if (d.each <= 1) return launch_route<T, 64, 1>(a, d, s);
    if (d.each <= 2) return launch_route<T, 64, 2>(a, d, s);
    if (d.each <= 4) return launch_route<T, 64, 4>(a, d, s);
    if (d.each <= 8) return launch_route<T, 64, 8>(a, d, s);
    if (d.each <= 16) return launch_route<T, 64, 16>(a, d, s);
    return launch_route<T, 64, 32>(a, d, s);
}

}  // namespace

hipError_t route(const RouteArgs& a, hipStream_t s) {
    if (a.counts != nullptr) {
        const hipError_t e = fill_i32(a.counts, a.nexperts, 0, s);
        if (e != hipSuccess) return e;
    }
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
