// C = beta*C + A*S with A in 8 bits (e4m3) and fp32 scales: A[i, r] = scales[i / group, r] * q[i, r].
//
// The gathers of A's columns bound A*S; codes are a quarter of the fp32 bytes. One wavefront owns a column of S. A column
// longer than a segment is cut at the multiples of the segment length in the array of nonzeros: its own wave goes up to the
// first of them, the wave of every multiple inside it takes the segment that begins there, found by a search in jc, and
// leaves a partial sum; these are added in order. Sums are fp32. A segment is an eighth of "seglen" nonzeros, so that no
// wave is still walking when the others are done (k = 1024, columns of power-law lengths up to 2000: 352 us at 128 nonzeros,
// 364 at 256, 470 at 1024), or a quarter where a wave takes eight nonzeros and more at a time (k = 64: 74 us at 256, 82 at 128).
// LPN lanes cover 16 * LPN rows with one 16-byte load each; a wave works on 64 / LPN nonzeros at a time.
//
// What bounds it: lines of A that miss L2, which come at 7.0 to 7.7 TB/s whatever lies behind it. k = 1024, 200000 columns
// of A, 2 M nonzeros in 50000 columns of 40: 350 us, 5.8 TB/s of gathers and 0.6 TB/s of C (one gather at a time 746 us;
// four in flight per lane as good as eight or sixteen, which cost occupancy where k is small). Rows of a column that
// different groups of lanes hold are added by exchanging halves (k = 16, 4 M nonzeros in 100000 columns: 51 us; with all 16
// sums shuffled through LDS 114 us). A small k takes a line for its codes and one for its scale per nonzero: 200000 columns
// of A, k = 64, 4 M nonzeros 77 us (13 TB/s of lines of 128 bytes; L2 holds part of the 13.6 MB of A), k = 100, 2 M 73 us (7.0 TB/s;
// 21 MB), k = 16, 4 M 60 us (17 TB/s; 4 MB). What the operands have, 72, 77 and 43 MB, would take 14, 15 and 9 us at a copy's rate.
#include "columns.hpp"
#include "common.hpp"
#include "kernels.hpp"
#include "workspace.hpp"
#include <algorithm>
#include <limits.h>

namespace bm {
namespace {

// Columns of S per launch, and segments at most: together they stay below 2^32 threads.
constexpr int kSlab = 1 << 24, kSegsMax = 1 << 25;
// Few nonzeros: segments are halved, down to kSegMin, until there are kWavesMin of them, since a wave's nonzeros follow one
// another with the whole way to memory (k = 612, 800 nonzeros in 63 columns of power-law lengths: 12 us, 28 with segments of
// 128; k = 1650, 4300 in 717: 17 and 60; for 2048 waves k = 1024, 2000 columns of 40: 27 against 20). Workgroups that add
// partial sums, at least as many, where there are so many columns.
constexpr int kSegMin = 16, kWavesMin = 1024, kLookWgs = 2048;
// Bytes of partial sums, at most: which columns are cut is known to the device alone, so that room is for every segment. Longer
// segments rather than more of it: 98 M nonzeros in 100000 columns, k = 256, take 3.20 ms with 256 MiB (segments of 376), 3.31 with
// the 0.8 GB of segments of 128; 9.9 M in 20000, k = 1024, 1.23 ms (152) and 1.25.
constexpr long long kPartialMax = 256LL << 20;

struct Q8Args {
    int k, ncols, nnz, seglen, beta, nscales, shift;      // shift: log2 of the rows per scale; 31: one scale per column
    int row0, row1;                                       // rows of this launch
    int nsegs;                                            // waves in front of the columns', one per multiple of seglen
    long long ldq;
    const unsigned char* Q;
    const float *scales, *vals;
    const int *ir, *jc;
    float *C, *partial;
};

typedef float f32x2 __attribute__((ext_vector_type(2)));

// Rows i .. i+15 of a column of k codes (i < k). A short last part is loaded as the column's last 16 codes, and shifted down
// by settle_codes when its turn comes: nothing between the loads waits for one of them.
__device__ __forceinline__ uint4 load_codes(const unsigned char* col, int i, int k) {
    uint4 x = make_uint4(0, 0, 0, 0);
    if (k >= 16) {
        const int s = i + 16 - k > 0 ? i + 16 - k : 0;          // codes in front of row i
        __builtin_memcpy(&x, col + i - s, 16);
    } else {
        unsigned w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < 15; ++j)
            if (i + j < k) w[j >> 2] |= (unsigned)col[i + j] << (8 * (j & 3));
        x = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return x;
}
__device__ __forceinline__ uint4 settle_codes(uint4 x, int i, int k) {
    if ((k & 15) == 0 || k < 16) return x;
    const int s = i + 16 - k > 0 ? i + 16 - k : 0;
    if (s & 8) x = make_uint4(x.z, x.w, 0, 0);
    if (s & 4) x = make_uint4(x.y, x.z, x.w, 0);
    x.x = __builtin_amdgcn_alignbyte(x.y, x.x, s & 3);
    x.y = __builtin_amdgcn_alignbyte(x.z, x.y, s & 3);
    x.z = __builtin_amdgcn_alignbyte(x.w, x.z, s & 3);
    x.w = __builtin_amdgcn_alignbyte(0u, x.w, s & 3);
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
            x[u] = load_codes(a.Q + r * a.ldq, i, a.k);
            by[u] = a.scales[r * a.nscales + sg];
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) fma_codes(acc, settle_codes(x[u], i, a.k), FULL || (it0 + u) * NG + g < rem ? v[u] * by[u] : 0.f);
}

// Segments begin at the multiples of seglen counted from the first nonzero, jc[0] (a range of columns may be passed with the
// whole matrix's arrays). The first one that begins at or after position x:
__device__ __forceinline__ int segment_from(const Q8Args& a, int x) { return (int)(((long long)x - a.jc[0] + a.seglen - 1) / a.seglen); }

// a summed over the two halves of the wave (HALVES) or over the two rows of 16 lanes of each half, in the lower of the two,
// and b in the upper one.
template <bool HALVES>
__device__ __forceinline__ float split_sum(float a, float b) {
    unsigned x = __float_as_uint(a), y = __float_as_uint(b);
    if constexpr (HALVES) {
        const auto r = __builtin_amdgcn_permlane32_swap(x, y, false, false);
        x = r[0]; y = r[1];
    } else {
        const auto r = __builtin_amdgcn_permlane16_swap(x, y, false, false);
        x = r[0]; y = r[1];
    }
    return __uint_as_float(x) + __uint_as_float(y);
}

// Rows i .. i+W-1 of a column of k sums, those past its end left out.
template <int W>
__device__ __forceinline__ void store_rows(float* col, int i, int k, const float (&v)[16], bool add) {
    if (i + W <= k) {
        float o[W];
        if (add) __builtin_memcpy(o, col + i, sizeof(o));
#pragma unroll
        for (int j = 0; j < W; ++j) o[j] = add ? o[j] + v[j] : v[j];
        __builtin_memcpy(col + i, o, sizeof(o));
    } else {
#pragma unroll
        for (int j = 0; j < W; ++j)
            if (i + j < k) col[i + j] = add ? col[i + j] + v[j] : v[j];
    }
}

// STAGED (LPN = 64): a lane's 16 rows go to C through LDS, so that a store covers one stretch of 1 KiB instead of 16 bytes of
// every 64.
template <int LPN, bool STAGED>
__global__ __launch_bounds__(BM_BLOCK) void k_dsmult_q8(Q8Args a) {
    constexpr int NG = 64 / LPN;
    __shared__ float stage[STAGED ? BM_WAVES_PER_BLOCK : 1][STAGED ? 16 * LPN : 1];
    const int lane = threadIdx.x & 63, l = lane % LPN, g = lane / LPN;
    const long long w = (long long)blockIdx.x * BM_WAVES_PER_BLOCK + wave_uniform(threadIdx.x >> 6);
    int lo, hi;
    float* out;
    bool add = false;
    if (w >= a.nsegs) {
        const long long c = w - a.nsegs;
        if (c >= a.ncols) return;
        lo = a.jc[c];
        hi = a.jc[c + 1];
        if (hi - lo > a.seglen) hi = a.jc[0] + segment_from(a, lo) * a.seglen;
        out = a.C + c * a.k;
        add = a.beta != 0;
    } else {
        const long long from = a.jc[0] + w * a.seglen;
        if (from >= a.jc[a.ncols]) return;
        lo = (int)from;
        int c0 = 0, c1 = a.ncols;                    // jc[c0] <= lo < jc[c1]
        while (c1 - c0 > 1) {
            const int mid = (int)(((long long)c0 + c1) >> 1);
            if (a.jc[mid] <= lo) c0 = mid; else c1 = mid;
        }
        const int end = a.jc[c1];
        if (end - a.jc[c0] <= a.seglen) return;      // its column's own wave takes all of it
        hi = end - lo > a.seglen ? lo + a.seglen : end;
        out = a.partial + w * a.k;
    }
    // (long columns of A: workgroups of their own for every 1024 rows, k = 2500, 10000 columns of 40: 228 us, one after another 276)
    for (long long from = a.row0 + (long long)blockIdx.y * 16 * LPN; from < a.row1; from += (long long)gridDim.y * 16 * LPN) {
        const int k0 = (int)from, i = k0 + 16 * l, left = a.k - i;
        const int sg = a.shift < 31 && left > 0 ? i >> a.shift : 0;
        float acc[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[j] = 0.f;
        constexpr int U = LPN < 4 ? LPN : 4;
        // (by what is left: hi may be the last int)
        for (int j0 = lo, after = hi - lo; after > 0; j0 = (int)(j0 + 64u), after -= 64) {
            const int rem = after < 64 ? after : 64;
            int row = 0;
            float val = 0.f;
            if (lane < rem) {
                row = a.ir[j0 + lane];
                val = a.vals[j0 + lane];
            }
            const int turns = (rem + NG - 1) / NG;         // per group
            int it = 0;
            for (; (it + U) * NG <= rem; it += U) gather_codes<LPN, U, true>(a, row, val, rem, it, g, i, left, sg, acc);
            for (; it < turns; it += U) gather_codes<LPN, U, false>(a, row, val, rem, it, g, i, left, sg, acc);
        }
        // the groups' sums: the wave's halves, then rows of 16 lanes exchange half of their rows of C (one exchange and one
        // addition give two sums), and what is left lies inside a row of lanes
        int off = 0;
        constexpr int W = NG == 1 ? 16 : NG == 2 ? 8 : 4;
        if constexpr (NG >= 2) {
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[j] = split_sum<true>(acc[j], acc[j + 8]);
            off += lane & 32 ? 8 : 0;
        }
        if constexpr (NG >= 4) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                acc[j] = split_sum<false>(acc[j], acc[j + 4]);
                if constexpr (LPN <= 8) acc[j] += dpp_mov<0x128>(acc[j]);      // row_ror 8, 4, 2, 1
                if constexpr (LPN <= 4) acc[j] += dpp_mov<0x124>(acc[j]);
                if constexpr (LPN <= 2) acc[j] += dpp_mov<0x122>(acc[j]);
                if constexpr (LPN <= 1) acc[j] += dpp_mov<0x121>(acc[j]);
            }
            off += lane & 16 ? 4 : 0;
        }
        if constexpr (STAGED) {
            float* mine = stage[threadIdx.x >> 6];
#pragma unroll
            for (int j = 0; j < W; j += 4)
                *(float4*)(mine + 16 * l + off + j) = make_float4(acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
            __builtin_amdgcn_wave_barrier();          // a wave's LDS operations take effect in order
#pragma unroll
            for (int j = 0; j < 16 * LPN; j += 256) {
                float v[16];
                *(float4*)v = *(const float4*)(mine + j + 4 * lane);
                if (k0 + j + 4 * lane < a.k) store_rows<4>(out, k0 + j + 4 * lane, a.k, v, add);
            }
            __builtin_amdgcn_wave_barrier();
        } else if (LPN >= 16 || (lane & 15) < LPN) {
            store_rows<W>(out, i + off, a.k, acc, add);
        }
    }
}

// C[:,c] += the partial sums of column c's segments, in order. A workgroup looks at `look` columns and adds those that were
// cut with all of its threads, W rows each (k = 1024: 15 us with four rows, 27 with one; k = 250: one is 2 us faster).
template <int W>
__global__ __launch_bounds__(BM_BLOCK) void k_add_segments(Q8Args a, int look) {
    const int lane = threadIdx.x & 63;
    const long long first = (long long)blockIdx.x * look;
    bool long_ = false;
    if (lane < look && first + lane < a.ncols) long_ = a.jc[first + lane + 1] - a.jc[first + lane] > a.seglen;
    for (unsigned long long cut = __ballot(long_); cut != 0; cut &= cut - 1) {
        const long long c = first + __builtin_ctzll(cut);
        const int s0 = segment_from(a, a.jc[c]);
        const int s1 = min(segment_from(a, a.jc[c + 1]), a.nsegs);
        for (int el = (int)threadIdx.x * W; el < a.k; el += BM_BLOCK * W) {
            const int rows = min(W, a.k - el);
            float acc[W];
            float* col = a.C + c * a.k + el;
            const float* part = a.partial + el;
            if (rows == W) {
                __builtin_memcpy(acc, col, sizeof(acc));
#pragma unroll 8
                for (int s = s0; s < s1; ++s) {
                    float p[W];
                    __builtin_memcpy(p, part + (long long)s * a.k, sizeof(p));
#pragma unroll
                    for (int j = 0; j < W; ++j) acc[j] += p[j];
                }
                __builtin_memcpy(col, acc, sizeof(acc));
            } else {
                for (int j = 0; j < rows; ++j) {
                    float x = col[j];
                    for (int s = s0; s < s1; ++s) x += part[(long long)s * a.k + j];
                    col[j] = x;
                }
            }
        }
    }
}

template <int LPN, bool STAGED = false>
hipError_t launch_q8(const Q8Args& a, long long nwaves, hipStream_t s) {
    hipLaunchKernelGGL((k_dsmult_q8<LPN, STAGED>), dim3((unsigned)((nwaves + BM_WAVES_PER_BLOCK - 1) / BM_WAVES_PER_BLOCK), (unsigned)std::min((a.row1 - a.row0 + 16LL * LPN - 1) / (16 * LPN), 65535LL)),
                       dim3(BM_BLOCK), 0, s, a);
    return hipGetLastError();
}

hipError_t q8_rows(const Q8Args& a, long long nwaves, hipStream_t s) {
    const int lanes = pow2ceil((a.row1 - a.row0 + 15) / 16);
    if (lanes <= 1) return launch_q8<1>(a, nwaves, s);
    if (lanes <= 2) return launch_q8<2>(a, nwaves, s);
    if (lanes <= 4) return launch_q8<4>(a, nwaves, s);
    if (lanes <= 8) return launch_q8<8>(a, nwaves, s);
    if (lanes <= 16) return launch_q8<16>(a, nwaves, s);
    if (lanes <= 32) return launch_q8<32>(a, nwaves, s);
    // Few nonzeros per column: C's stores are what counts (k = 1024, 100000 columns of 2: 123 us staged, 158 not; of 8: 204 and
    // 223). With more, the gathers do, and they run faster beside the scattered stores (of 16: 329 and 319; 50000 of 32: 297 and 291).
    if (a.nnz < 12LL * a.ncols) return launch_q8<64, true>(a, nwaves, s);
    return launch_q8<64>(a, nwaves, s);
}

}  // namespace

hipError_t dsmult_q8_csc(int k, int ncols, int nnz, const unsigned char* Q, long long ldq, const float* scales, int group,
                         const float* vals, const int* ir, const int* jc, float* C, int beta, hipStream_t s) {
    for (; ncols > kSlab; ncols -= kSlab, jc += kSlab, C += (long long)kSlab * k) {
        const hipError_t e = dsmult_q8_csc(k, kSlab, nnz, Q, ldq, scales, group, vals, ir, jc, C, beta, s);
        if (e != hipSuccess) return e;
    }
    Q8Args a;
    a.k = k; a.ncols = ncols; a.nnz = nnz; a.beta = beta;
    a.seglen = std::max(opt_seglen() / (k > 128 ? 8 : 4), nnz / kSegsMax + 1);
    a.nscales = group == 0 ? 1 : (k + group - 1) / group;
    a.shift = group == 0 ? 31 : group == 32 ? 5 : group == 64 ? 6 : 7;
    a.ldq = ldq; a.Q = Q; a.scales = scales; a.vals = vals; a.ir = ir; a.jc = jc; a.C = C;
    a.partial = nullptr;
    a.nsegs = 0;
    hipError_t err;
    while (a.seglen > kSegMin && nnz < kWavesMin * (long long)a.seglen) a.seglen >>= 1;
    const long long most = kPartialMax / ((long long)sizeof(float) * k);          // segments
    if (nnz > most * a.seglen) a.seglen = most > 0 ? (int)((nnz + most - 1) / most) : INT_MAX;
    if (nnz > a.seglen) {
        a.nsegs = (int)((nnz + (long long)a.seglen - 1) / a.seglen);
        a.partial = (float*)ws_get(WS_PARTIAL, sizeof(float) * (size_t)a.nsegs * (size_t)k, &err, s);
        if (!a.partial) return err;
    }
    const long long nwaves = (long long)ncols + a.nsegs;
    // Up to 256 rows past a multiple of 1024, which would leave most of a wave without work, get a launch of their own with fewer
    // lanes per nonzero (600000 nonzeros, k = 1025: 152 us instead of 175, k = 1280: 155 and 164; more rows lose: 1500: 203 and 196),
    // where the nonzeros are worth one (1500 nonzeros, k = 1056: 15 us, in one launch 12).
    const int tail = k > 1024 && k % 1024 <= 256 && nnz >= (1 << 16) ? k % 1024 : 0;
    a.row0 = 0;
    a.row1 = k - tail;
    err = q8_rows(a, nwaves, s);
    if (err == hipSuccess && tail > 0) {
        a.row0 = k - tail;
        a.row1 = k;
        err = q8_rows(a, nwaves, s);
    }
    if (err == hipSuccess && a.nsegs > 0) {
        const int look = std::min(std::max(ncols / kLookWgs, 1), 16);
        hipLaunchKernelGGL((k > BM_BLOCK ? k_add_segments<4> : k_add_segments<1>), dim3((unsigned)((ncols + look - 1LL) / look)), dim3(BM_BLOCK), 0, s, a, look);
        err = hipGetLastError();
    }
    return err;
}

}  // namespace bm
