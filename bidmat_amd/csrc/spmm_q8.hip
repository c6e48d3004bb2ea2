// C = beta*C + A*S with A in 8 bits (e4m3) and fp32 scales: A[i, r] = scales[i / group, r] * q[i, r].
//
// The gathers of A's columns bound A*S; codes are a quarter of the fp32 bytes. One wavefront owns a column of S, like in
// the fp32 product (spmm.hip), with its rule for long columns: a column longer than "seglen" nonzeros is cut, extra waves
// take the other segments and leave partial sums that are added in order. Sums are fp32.
// LPN lanes cover 16 * LPN rows with one 16-byte load each; a wave works on 64 / LPN nonzeros at a time.
#include "columns.hpp"
#include "common.hpp"
#include "kernels.hpp"
#include "workspace.hpp"

namespace bm {
namespace {

struct Q8Args {
    int k, ncols, seglen, beta, nscales, shift;      // shift: log2 of the rows per scale; 31: one scale per column
    long long ldq;
    const unsigned char* Q;
    const float *scales, *vals;
    const int *ir, *jc, *ovf;
    float *C, *partial;
};

typedef float f32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ uint4 load_codes(const unsigned char* p, int left) {
    uint4 x = make_uint4(0, 0, 0, 0);
    if (left >= 16) {
        __builtin_memcpy(&x, p, 16);
    } else {
        unsigned w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < 16; ++j)
            if (j < left) w[j >> 2] |= (unsigned)p[j] << (8 * (j & 3));
        x = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return x;
}
__device__ __forceinline__ void fma_codes(float (&acc)[16], uint4 x, float by) {
    const unsigned w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], false);
        const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], true);
        acc[4 * i] = fmaf(lo.x, by, acc[4 * i]);
        acc[4 * i + 1] = fmaf(lo.y, by, acc[4 * i + 1]);
        acc[4 * i + 2] = fmaf(hi.x, by, acc[4 * i + 2]);
        acc[4 * i + 3] = fmaf(hi.y, by, acc[4 * i + 3]);
    }
}

// Nonzeros it0 .. it0 + U - 1 of every group (slot it * NG + g of the wave's chunk of 64, held one per lane): U gathers in
// flight per lane before their sums are taken. FULL: all of them exist.
template <int LPN, int U, bool FULL>
__device__ __forceinline__ void gather_codes(const Q8Args& a, int row, float val, int rem, int it0, int g, int i, int left, int sg, float (&acc)[16]) {
    constexpr int NG = 64 / LPN;
    uint4 x[U];
    float by[U], v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int src = (it0 + u) * NG + g;
        long long r;
        if constexpr (LPN == 64) {
            r = __builtin_amdgcn_readlane(row, it0 + u);
            v[u] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(val), it0 + u));
        } else {
            r = lane_read(row, src);
            v[u] = lane_read(val, src);
        }
        by[u] = 0.f;
        x[u] = make_uint4(0, 0, 0, 0);
        if (left > 0 && (FULL || src < rem)) {
            x[u] = load_codes(a.Q + r * a.ldq + i, left);
            by[u] = a.scales[r * a.nscales + sg];
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) fma_codes(acc, x[u], FULL || (it0 + u) * NG + g < rem ? v[u] * by[u] : 0.f);
}

template <int LPN>
__global__ __launch_bounds__(BM_BLOCK) void k_dsmult_q8(Q8Args a) {
    constexpr int NG = 64 / LPN;
    const int lane = threadIdx.x & 63, l = lane % LPN, g = lane / LPN;
    const long long w = (long long)blockIdx.x * BM_WAVES_PER_BLOCK + wave_uniform(threadIdx.x >> 6);
    int lo, hi;
    float* out;
    bool add = false;
    if (w < a.ncols) {
        lo = a.jc[w];
        hi = a.jc[w + 1];
        if (hi - lo > a.seglen) hi = lo + a.seglen;
        out = a.C + w * a.k;
        add = a.beta != 0;
    } else {
        if (a.ovf == nullptr) return;
        const long long x = w - a.ncols;
        if (x >= a.ovf[a.ncols]) return;
        int c0 = 0, c1 = a.ncols;                    // ovf[c0] <= x < ovf[c1]
        while (c1 - c0 > 1) {
            const int mid = (int)(((long long)c0 + c1) >> 1);
            if (a.ovf[mid] <= x) c0 = mid; else c1 = mid;
        }
        const long long from = (long long)a.jc[c0] + (x - a.ovf[c0] + 1) * a.seglen, end = a.jc[c0 + 1];
        lo = (int)from;
        hi = (int)(end < from + a.seglen ? end : from + a.seglen);
        out = a.partial + x * a.k;
    }
    for (int k0 = 0; k0 < a.k; k0 += 16 * LPN) {
        const int i = k0 + 16 * l, left = a.k - i;
        const int sg = a.shift < 31 && left > 0 ? i >> a.shift : 0;
        float acc[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[j] = 0.f;
        constexpr int U = LPN < 8 ? LPN : 8;
        for (int j0 = lo; j0 < hi; j0 += 64) {
            const int rem = hi - j0 < 64 ? hi - j0 : 64;
            int row = 0;
            float val = 0.f;
            if (lane < rem) {
                row = a.ir[j0 + lane];
                val = a.vals[j0 + lane];
            }
            const int turns = (rem + NG - 1) / NG;         // per group
            int it = 0;
            for (; (it + U) * NG <= rem; it += U) gather_codes<LPN, U, true>(a, row, val, rem, it, g, i, left, sg, acc);
            for (; it < turns; it += (U > 4 ? 4 : U)) gather_codes<LPN, (U > 4 ? 4 : U), false>(a, row, val, rem, it, g, i, left, sg, acc);
        }
#pragma unroll
        for (int m = LPN; m < 64; m <<= 1)
#pragma unroll
            for (int j = 0; j < 16; ++j) acc[j] += __shfl_xor(acc[j], m, 64);
        if (g == 0) {
            if (left >= 16) {
                float4 o[4];
                if (add) __builtin_memcpy(o, out + i, 64);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float4 s = make_float4(acc[4 * j], acc[4 * j + 1], acc[4 * j + 2], acc[4 * j + 3]);
                    o[j] = add ? make_float4(o[j].x + s.x, o[j].y + s.y, o[j].z + s.z, o[j].w + s.w) : s;
                }
                __builtin_memcpy(out + i, o, 64);
            } else {
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    if (j < left) out[i + j] = add ? out[i + j] + acc[j] : acc[j];
            }
        }
    }
}

template <int LPN>
hipError_t launch_q8(const Q8Args& a, long long nwaves, hipStream_t s) {
    hipLaunchKernelGGL((k_dsmult_q8<LPN>), dim3((unsigned)((nwaves + BM_WAVES_PER_BLOCK - 1) / BM_WAVES_PER_BLOCK)), dim3(BM_BLOCK), 0, s, a);
    return hipGetLastError();
}

}  // namespace

hipError_t dsmult_q8_csc(int k, int ncols, int nnz, const unsigned char* Q, long long ldq, const float* scales, int group,
                         const float* vals, const int* ir, const int* jc, float* C, int beta, hipStream_t s) {
    Q8Args a;
    a.k = k; a.ncols = ncols; a.seglen = opt_seglen(); a.beta = beta;
    a.nscales = group == 0 ? 1 : (k + group - 1) / group;
    a.shift = group == 0 ? 31 : group == 32 ? 5 : group == 64 ? 6 : 7;
    a.ldq = ldq; a.Q = Q; a.scales = scales; a.vals = vals; a.ir = ir; a.jc = jc; a.C = C;
    a.ovf = nullptr; a.partial = nullptr;
    int* ovf = nullptr;
    hipError_t err = build_overflow_table(ncols, nnz, jc, a.seglen, &ovf, s);
    if (err != hipSuccess) return err;
    long long extra = 0;
    if (ovf != nullptr) {
        extra = nnz / a.seglen;
        a.ovf = ovf;
        a.partial = (float*)ws_get(WS_PARTIAL, sizeof(float) * (size_t)extra * (size_t)k, &err, s);
        if (!a.partial) return err;
    }
    const long long nwaves = (long long)ncols + extra;
    const int lanes = pow2ceil((k + 15) / 16);
    if (lanes <= 1) err = launch_q8<1>(a, nwaves, s);
    else if (lanes <= 2) err = launch_q8<2>(a, nwaves, s);
    else if (lanes <= 4) err = launch_q8<4>(a, nwaves, s);
    else if (lanes <= 8) err = launch_q8<8>(a, nwaves, s);
    else if (lanes <= 16) err = launch_q8<16>(a, nwaves, s);
    else if (lanes <= 32) err = launch_q8<32>(a, nwaves, s);
    else err = launch_q8<64>(a, nwaves, s);
    if (err == hipSuccess && ovf != nullptr) err = overflow_reduce(k, ncols, ovf, a.partial, C, s);
    return err;
}

}  // namespace bm
