// Root-mean-square normalisation of the columns of a dense matrix, with the residual's addition in front, an output in
// 8 bits with scales behind, and its gradient.
//
//   h = x + r,   rs = 1 / sqrt(mean(h^2) + eps),   y_i = h_i * rs * w_i
//   scale_g = max(max over group g of |y| / 448, 2^-126),   q_i = e4m3(y_i / scale_g)
//
// y is formed from the sum in fp32, not from the rounded h that is written. 448 is the largest number of e4m3, so that no
// code overflows; 2^-126 keeps 1 / scale finite for a group of zeros (whose codes are zeros).
// TPC threads share a column and keep all of it in registers (8 * NV elements each): every input is read once and every
// output written once, also where an output overwrites its input.
//
// What bounds it: memory, as long as columns of a multiple of 128 bytes let every load take whole lines (8192 rows x 16384
// columns bf16 with residual and codes: 160 us, 5.9 TB/s). Odd heights: 1001 x 155540 bf16, read and written, 120 us, 5.2 TB/s; 1001
// x 77777 fp32, with codes too, 141 us, 5.0. A tenth of these columns stays in the 256 MB cache, which is no faster here (13.7
// us, 4.5 TB/s and 13.5 us, 5.2, in a run of calls; a dispatch of the latter by itself 17.5): the start and the end of a
// launch of 14 us are most of what is lost against the cache's 8. A few columns: the launch. A workgroup of its own per
// column from 1025 rows on, more than one column per wave up to 256.
#include "columns.hpp"
#include "elems.hpp"
#include "kernels.hpp"
#include "workspace.hpp"

namespace bm {
namespace {

constexpr float kE4M3Max = 448.f;
constexpr float kScaleMin = 1.17549435e-38f;      // 2^-126

constexpr int norm_block(int tpc) { return tpc <= 64 ? BM_BLOCK : tpc; }

__device__ __forceinline__ float square_sum(float8_t x) {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) s = fmaf(x[j], x[j], s);
    return s;
}
__device__ __forceinline__ float abs_max(float8_t x) {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) s = fmaxf(s, fabsf(x[j]));
    return s;
}

// The sum of a column's squares may leave fp32 on either side: d = mean(h^2) + eps is infinite, or so small (below 2^-126) that
// squares which count in it have few digits or vanished. It is taken again from h * by * rest = h * 2^-96 or h * 2^96, whose
// squares and their sums stay inside for every h of fp32, and y = (h * by) * rs * w: with h of the largest values half of the
// factor stays with rs, so that neither it nor h * by has few digits. (An infinite h leaves rs = 0.)
__device__ __forceinline__ bool in_range(float d) { return d >= 0x1p-126f && d < INFINITY; }
struct Rescale {
    float by, rest;
    __device__ __forceinline__ float rs(float mean, float eps) const { return rest / sqrtf(mean + eps * (by * rest) * (by * rest)); }
};
__device__ __forceinline__ Rescale rescale(float d) { return d < 1.f ? Rescale{0x1p96f, 1.f} : Rescale{0x1p-48f, 0x1p-48f}; }

// Eight e4m3 codes (OCP, round to nearest even).
__device__ __forceinline__ uint2 e4m3_codes(float8_t x) {
    int a = 0, b = 0;
    a = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], a, false);
    a = __builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], a, true);
    b = __builtin_amdgcn_cvt_pk_fp8_f32(x[4], x[5], b, false);
    b = __builtin_amdgcn_cvt_pk_fp8_f32(x[6], x[7], b, true);
    return make_uint2((unsigned)a, (unsigned)b);
}
__device__ __forceinline__ void store_codes(unsigned char* col, int i, int n, uint2 c) {
    if (i + 8 <= n) { __builtin_memcpy(col + i, &c, 8); return; }
    const unsigned long long bits = c.x | ((unsigned long long)c.y << 32);
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (i + j < n) col[i + j] = (unsigned char)(bits >> (8 * j));
}

// Largest value over the lanes of one group of rows (group / 8 lanes, or fewer when the column has fewer).
__device__ __forceinline__ float lanes_allmax(float x, int lanes) {
    if (lanes >= 2) x = fmaxf(x, dpp_mov<DPP_QUAD_XOR1>(x));
    if (lanes >= 4) x = fmaxf(x, dpp_mov<DPP_QUAD_XOR2>(x));
    if (lanes >= 8) x = fmaxf(x, dpp_mov<DPP_ROW_HALF_MIRROR>(x));
    if (lanes >= 16) x = fmaxf(x, dpp_mov<DPP_ROW_MIRROR>(x));
    return x;
}

template <class T, int TPC, int NV, bool RAGGED>
__global__ __launch_bounds__(norm_block(TPC)) void k_rmsnorm(NormArgs a) {
    constexpr int CPB = norm_block(TPC) / TPC;
    __shared__ float sh[3][TPC > 64 ? TPC / 64 : 1];
    const long long c = (long long)blockIdx.x * CPB + threadIdx.x / TPC;
    if (c >= a.ncols) return;
    const int t = threadIdx.x % TPC, n = a.nrows;
    const T* x = (const T*)a.X + c * a.ldx;
    // (whole heights go through load_col8 too, whose branches keep a wave from asking for everything at once: 8192 rows x 16384
    // columns bf16 160 us, without them 165)
    auto load = [&](const auto* col, int v) {
        if constexpr (RAGGED) return fetch_col8<true>(col, (v * TPC + t) * 8, n);
        else return load_col8(col, (v * TPC + t) * 8, n);
    };
    auto settle = [&](auto part, int v) { return settle_col8<RAGGED>(part, (v * TPC + t) * 8, n).wide(); };
    float8_t h[NV];
    if (RAGGED && a.R != nullptr) {
        const T* r = (const T*)a.R + c * a.ldr;
        Raw8<T> xs[NV], rs[NV];
#pragma unroll
        for (int v = 0; v < NV; ++v) { xs[v] = load(x, v); rs[v] = load(r, v); }
#pragma unroll
        for (int v = 0; v < NV; ++v) h[v] = settle(xs[v], v) + settle(rs[v], v);
    } else {
#pragma unroll
        for (int v = 0; v < NV; ++v) h[v] = settle(load(x, v), v);
        if (a.R != nullptr) {
            const T* r = (const T*)a.R + c * a.ldr;
#pragma unroll
            for (int v = 0; v < NV; ++v) h[v] += settle(load(r, v), v);
        }
    }
    float ss = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) ss += square_sum(h[v]);
    if (a.H != nullptr) {
        T* o = (T*)a.H + c * a.ldh;
#pragma unroll
        for (int v = 0; v < NV; ++v) store_col8(o, (v * TPC + t) * 8, n, h[v]);
    }
    if (a.Y == nullptr && a.Q == nullptr) return;
    ss = column_allsum<TPC>(ss, sh[0]);
    const float d = ss / (float)n + a.eps;
    float rs = 1.f / sqrtf(d);
    if (!in_range(d)) {
        const Rescale r = rescale(d);
        float sum = 0.f;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            h[v] = h[v] * r.by;
            sum += square_sum(h[v] * r.rest);
        }
        rs = r.rs(column_allsum<TPC>(sum, sh[2]) / (float)n, a.eps);
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        h[v] = h[v] * rs * settle(load(a.w, v), v);
    }
    if (a.Y != nullptr) {
        T* o = (T*)a.Y + c * a.ldy;
#pragma unroll
        for (int v = 0; v < NV; ++v) store_col8(o, (v * TPC + t) * 8, n, h[v]);
    }
    if (a.Q == nullptr) return;
    unsigned char* q = a.Q + c * a.ldq;
    if (a.group == 0) {
        float m = 0.f;
#pragma unroll
        for (int v = 0; v < NV; ++v) m = fmaxf(m, abs_max(h[v]));
        m = column_allmax<TPC>(m, sh[1]);
        const float scale = fmaxf(m / kE4M3Max, kScaleMin), inv = 1.f / scale;
        if (t == 0) a.scales[c] = scale;
#pragma unroll
        for (int v = 0; v < NV; ++v) store_codes(q, (v * TPC + t) * 8, n, e4m3_codes(h[v] * inv));
        return;
    }
    const int lanes = a.group >> 3, ng = (n + a.group - 1) / a.group;
    const int span = lanes < TPC ? lanes : TPC;          // TPC < lanes: the column is one group
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int i = (v * TPC + t) * 8;
        const float m = lanes_allmax(abs_max(h[v]), span);
        const float scale = fmaxf(m / kE4M3Max, kScaleMin), inv = 1.f / scale;
        if (i < n) {
            if ((t & (span - 1)) == 0) a.scales[c * ng + i / a.group] = scale;
            store_codes(q, i, n, e4m3_codes(h[v] * inv));
        }
    }
}

// Gradients. With g = dy * w (elementwise) and u = h * rs:
//   dx = rs * (g - u * mean(g * u)) + dh,   dw_i = sum over columns of dy_i * u_i
// Every workgroup walks columns c0, c0 + slots, ... and keeps its share of dw in registers; the shares go to partial
// (one row of nrows floats per workgroup) and are added in a fixed order by k_add_shares.
// What bounds it: memory (4096 rows x 16384 columns bf16: 103 us with the shares' addition, 5.2 TB/s). Above 8192 rows a
// thread's registers do not hold the next column, above 16384 not the present one either (16384 rows x 4096: 118 us, 4.5 TB/s;
// 32768 x 2048: 202 us, 2.7 TB/s, spilling). Medium sizes: the shares and the second launch (1001 x 15554 bf16: 31 us for 93 MB,
// 37 with dH; 8192 x 2000: 27 us for 98 MB).
// A column whose sums leave fp32, of squares or of products (which count on the small side where rs is large).
__device__ __forceinline__ bool outside(float d, float gh) {
    return !in_range(d) || !(fabsf(gh) < INFINITY) || (d < 0x1p-20f && fabsf(gh) < 0x1p-100f);
}
// Those among a workgroup's columns, by the marks that the loop over all of them left: with u = h * by * rs, which is at most
// sqrt(n), and the mean of g * u. They are read again behind the others, which so keep their registers (within that loop this
// cost heights above 16384 12 to 46 %), and their part of dw is added to the share in memory, one column after the other.
template <class T, int TPC, int NV, bool RAGGED>
__device__ __forceinline__ void odd_columns(const NormGradArgs& a, float* share, const unsigned char* marks, float (*sh)[4][TPC > 64 ? TPC / 64 : 1]) {
    constexpr int CPB = norm_block(TPC) / TPC;
    const int t = threadIdx.x % TPC, n = a.nrows;
    int turn = 0;
    for (long long c0 = (long long)blockIdx.x * CPB; c0 < a.ncols; c0 += (long long)gridDim.x * CPB, marks += CPB)
        for (int q = 0; q < CPB; ++q) {
            const long long c = c0 + q;
            if (c >= a.ncols || marks[q] == 0) continue;          // the same for all threads of the workgroup
            if (threadIdx.x / TPC == q) {
                auto part = [&](const auto* col, int v) {
                    return settle_col8<RAGGED>(fetch_col8<RAGGED>(col, (v * TPC + t) * 8, n), (v * TPC + t) * 8, n).wide();
                };
                const T *h = (const T*)a.H + c * a.ldh, *dy = (const T*)a.dY + c * a.lddy;
                float sum = 0.f, by = 1.f, mean = 0.f;
#pragma unroll 1
                for (int v = 0; v < NV; ++v) sum += square_sum(part(h, v));
                const float d2 = column_allsum<TPC>(sum, sh[turn][0]) / (float)n + a.eps;
                float rs = 1.f / sqrtf(d2);
                if (!in_range(d2)) {
                    const Rescale r = rescale(d2);
                    by = r.by;
                    sum = 0.f;
#pragma unroll 1
                    for (int v = 0; v < NV; ++v) sum += square_sum(part(h, v) * by * r.rest);
                    rs = r.rs(column_allsum<TPC>(sum, sh[turn][1]) / (float)n, a.eps);
                }
#pragma unroll 1
                for (int v = 0; v < NV; ++v) {
                    const float8_t u = part(h, v) * by * rs * (1.f / (float)n), g = part(dy, v) * part(a.w, v);
#pragma unroll
                    for (int j = 0; j < 8; ++j) mean = fmaf(u[j], g[j], mean);
                }
                mean = column_allsum<TPC>(mean, sh[turn][2]);
#pragma unroll 1
                for (int v = 0; v < NV; ++v) {
                    const int i = (v * TPC + t) * 8;
                    const float8_t u = part(h, v) * by * rs, y = part(dy, v);
                    float8_t d = rs * (y * part(a.w, v) - u * mean) * by;
                    if (a.dH != nullptr) d += part((const T*)a.dH + c * a.lddh, v);
                    put_col8<RAGGED>((T*)a.dX + c * a.lddx, i, n, d);
                    if (share != nullptr) store_col8(share, i, n, load_col8(share, i, n).wide() + y * u);
                }
            }
            turn ^= 1;
            if constexpr (CPB > 1) __syncthreads();
        }
}

// Columns of one launch, per workgroup at most: a byte marks each of them (LDS).
constexpr int kNormMarks = 8192;

template <class T, int TPC, int NV, bool RAGGED>
__global__ __launch_bounds__(norm_block(TPC), 4) void k_rmsnorm_grad(NormGradArgs a, float* partial) {
    constexpr int CPB = norm_block(TPC) / TPC;
    __shared__ float sh[2][4][TPC > 64 ? TPC / 64 : 1];
    __shared__ unsigned char marks[kNormMarks];
    const int t = threadIdx.x % TPC, n = a.nrows;
    float8_t dw[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) dw[v] = (float8_t)(0.f);
    int turn = 0;
    bool odd = false;          // a column was left to odd_columns
    unsigned char* mark = marks + threadIdx.x / TPC;
    // A column's data are requested while the one before is worked on, where a thread's registers hold both.
    constexpr bool AHEAD = TPC < 1024 || NV == 1;
    const long long step = (long long)gridDim.x * CPB;
    long long c = (long long)blockIdx.x * CPB + threadIdx.x / TPC;
    Raw8<T> h[NV], g[NV], r[NV];
    auto fetch = [&](long long col) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            h[v] = fetch_col8<RAGGED>((const T*)a.H + col * a.ldh, (v * TPC + t) * 8, n);
            g[v] = fetch_col8<RAGGED>((const T*)a.dY + col * a.lddy, (v * TPC + t) * 8, n);
            if (AHEAD && a.dH != nullptr) r[v] = fetch_col8<RAGGED>((const T*)a.dH + col * a.lddh, (v * TPC + t) * 8, n);
        }
    };
    auto weight = [&](int v) { return settle_col8<RAGGED>(fetch_col8<RAGGED>(a.w, (v * TPC + t) * 8, n), (v * TPC + t) * 8, n).wide(); };
    float8_t w[NV];
    if (AHEAD) {
#pragma unroll
        for (int v = 0; v < NV; ++v) w[v] = weight(v);
    }
    if (AHEAD && c < a.ncols) fetch(c);
    for (; c < a.ncols; c += step) {
        if (!AHEAD) fetch(c);
        Raw8<T> hc[NV], gc[NV], rc[NV];
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int i = (v * TPC + t) * 8;
            hc[v] = settle_col8<RAGGED>(h[v], i, n);
            gc[v] = settle_col8<RAGGED>(g[v], i, n);
            if (AHEAD && a.dH != nullptr) rc[v] = settle_col8<RAGGED>(r[v], i, n);
        }
        if (AHEAD && c + step < a.ncols) fetch(c + step);
        float hh = 0.f, gh = 0.f;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const float8_t x = hc[v].wide(), y = gc[v].wide() * (AHEAD ? w[v] : weight(v));
            hh += square_sum(x);
#pragma unroll
            for (int j = 0; j < 8; ++j) gh = fmaf(x[j], y[j], gh);
        }
        hh = column_allsum<TPC>(hh, sh[turn][0]);
        const float d2 = hh / (float)n + a.eps, rs = 1.f / sqrtf(d2);
        gh = column_allsum<TPC>(gh, sh[turn][1]);
        const float mean = gh / (float)n * rs;          // of g * u
        const bool out = outside(d2, gh);
        if (t == 0) *mark = out;
        mark += CPB;
        if (TPC >= 64 ? __ballot(out) != 0 : out) {
            odd = true;
        } else {
            T* o = (T*)a.dX + c * a.lddx;
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const int i = (v * TPC + t) * 8;
                const float8_t u = hc[v].wide() * rs, y = gc[v].wide();
                float8_t d = rs * (y * (AHEAD ? w[v] : weight(v)) - u * mean);
                dw[v] += y * u;
                if (a.dH != nullptr) d += AHEAD ? rc[v].wide() : settle_col8<RAGGED>(fetch_col8<RAGGED>((const T*)a.dH + c * a.lddh, i, n), i, n).wide();
                put_col8<RAGGED>(o, i, n, d);
            }
        }
        turn ^= 1;
    }
    // a single workgroup's share is the gradient (partial == nullptr)
    float* share = a.dw == nullptr ? nullptr : partial != nullptr ? partial + (size_t)blockIdx.x * n : a.dw;
    const bool add = partial == nullptr && a.beta != 0;
    if (share != nullptr) {
        if constexpr (CPB > 1) {
            // the columns of a wave first, then the workgroup's four waves
            __shared__ float sum[BM_WAVES_PER_BLOCK][TPC * 8 * NV];
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    float d = dw[v][j];
#pragma unroll
                    for (int m = TPC; m < 64; m <<= 1) d += __shfl_xor(d, m, 64);
                    if ((threadIdx.x & 63) < TPC) sum[threadIdx.x >> 6][(v * TPC + t) * 8 + j] = d;
                }
            __syncthreads();
            for (int i = threadIdx.x; i < n; i += BM_BLOCK) {
                const float d = (sum[0][i] + sum[1][i]) + (sum[2][i] + sum[3][i]);
                share[i] = add ? share[i] + d : d;
            }
        } else {
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const int i = (v * TPC + t) * 8;
                store_col8(share, i, n, add ? load_col8(share, i, n).wide() + dw[v] : dw[v]);
            }
        }
    }
    if (__syncthreads_or(odd)) odd_columns<T, TPC, NV, RAGGED>(a, share, marks, sh);
}

// dw[i] = beta * dw[i] + sum over shares of partial[share][i]: 16 rows x 64 threads per workgroup; thread (x, y) adds every 64th
// share of row x, then the sums of a row are added by halves. (4 rows x 256 threads take longer at all heights with many shares:
// the whole gradient of 1000 rows x 15000 columns bf16 32.3 us against 27.6, 4096 x 16384 110 against 102; 256 x 4000 8.1 against 9.0.)
__global__ __launch_bounds__(1024) void k_add_shares(int n, int nshares, const float* __restrict__ partial, float* __restrict__ dw,
                                                     int beta) {
    constexpr int ROWS = 16, Y = 1024 / ROWS;
    __shared__ float sh[Y][ROWS + 1];
    const int x = threadIdx.x % ROWS, y = threadIdx.x / ROWS;
    const int i = blockIdx.x * ROWS + x;
    float s = 0.f;
    if (i < n) {
#pragma unroll 8
        for (int p = y; p < nshares; p += Y) s += partial[(size_t)p * n + i];
    }
    sh[y][x] = s;
    for (int step = Y / 2; step > 0; step >>= 1) {
        __syncthreads();
        if (y < step) sh[y][x] += sh[y + step][x];
    }
    if (y == 0 && i < n) dw[i] = beta ? dw[i] + sh[0][x] : sh[0][x];
}

template <class T, int TPC, int NV>
hipError_t launch_norm(const NormArgs& a, hipStream_t s) {
    constexpr int CPB = norm_block(TPC) / TPC;
    const unsigned grid = (unsigned)((a.ncols + CPB - 1LL) / CPB);
    hipLaunchKernelGGL((a.nrows % 8 != 0 ? k_rmsnorm<T, TPC, NV, true> : k_rmsnorm<T, TPC, NV, false>), dim3(grid), dim3(norm_block(TPC)), 0, s, a);
    return hipGetLastError();
}
// Workgroups of the gradient, at most: 16 waves per CU. More of them hide more latency but leave more shares of dw (4096
// rows x 16384 columns bf16: 256 workgroups of 512 threads 134 us, 512 113 us, 1024 116 us).
constexpr int norm_shares(int block) { return 262144 / block; }
template <class T, int TPC, int NV>
hipError_t launch_norm_grad(const NormGradArgs& a, hipStream_t s) {
    constexpr int CPB = norm_block(TPC) / TPC;
    const long long want = (a.ncols + CPB - 1LL) / CPB, most = norm_shares(norm_block(TPC));
    // up to four turns of one workgroup take less time than a second launch
    const unsigned grid = (unsigned)(a.dw != nullptr && want <= 4 ? 1 : want < most ? want : most);
    float* partial = nullptr;
    if (a.dw != nullptr && grid > 1) {
        hipError_t err;
        partial = (float*)ws_get(WS_NORM_SHARES, sizeof(float) * (size_t)grid * (size_t)a.nrows, &err, s);
        if (!partial) return err;
    }
    hipLaunchKernelGGL((a.nrows % 8 != 0 ? k_rmsnorm_grad<T, TPC, NV, true> : k_rmsnorm_grad<T, TPC, NV, false>), dim3(grid), dim3(norm_block(TPC)), 0, s, a, partial);
    if (a.dw != nullptr && grid > 1)
        hipLaunchKernelGGL(k_add_shares, dim3((a.nrows + 15) / 16), dim3(1024), 0, s, a.nrows, (int)grid, partial, a.dw, a.beta);
    return hipGetLastError();
}

// Threads per column and vectors per thread: the fewest that hold n elements. Forward, two vectors per thread cost little (4096
// rows x 16384 columns bf16 with residual 92.4 us, with 512 threads of one vector 89.7; 1000 x 15000 18.7 and 20.0; 768 x 20000 19.8
// and 19.0). The gradient keeps two or three columns at once, and one vector per thread leaves it registers (4096 x 16384 bf16
// 102 us, with 256 threads of two 123; 8192 x 8192 102 and 177; 1024 x 32768 fp32 108 and 281; 45 and 148 for 1000 x 15000;
// in 16 bits 128 threads are as good as 64 of two, 27.6 and 26.4).
template <class T, class F>
hipError_t by_height(int n, F&& f) {
    const int vecs = (n + 7) / 8;
    if (vecs <= 8) return f.template go<T, 8, 1>();
    if (vecs <= 16) return f.template go<T, 16, 1>();
    if (vecs <= 32) return f.template go<T, 32, 1>();
    if (vecs <= 64) return f.template go<T, 64, 1>();
    if (vecs <= 128) return f.template go<T, 64, 2>();
    if (vecs <= 256) return f.template go<T, 256, 1>();
    if (vecs <= 512) return f.template go<T, 256, 2>();
    if (vecs <= 1024) return f.template go<T, 512, 2>();
    if (vecs <= 2048) return f.template go<T, 1024, 2>();
    return f.template go<T, 1024, 4>();
}
template <class T, class F>
hipError_t by_height_grad(int n, F&& f) {
    const int vecs = (n + 7) / 8;
    if (vecs <= 8) return f.template go<T, 8, 1>();
    if (vecs <= 16) return f.template go<T, 16, 1>();
    if (vecs <= 32) return f.template go<T, 32, 1>();
    if (vecs <= 64) return f.template go<T, 64, 1>();
    if (vecs <= 128) return f.template go<T, 128, 1>();
    if (vecs <= 256) return f.template go<T, 256, 1>();
    if (vecs <= 512) return f.template go<T, 512, 1>();
    if (vecs <= 1024) return f.template go<T, 1024, 1>();
    if (vecs <= 2048) return f.template go<T, 1024, 2>();
    return f.template go<T, 1024, 4>();
}
struct Norm {
    const NormArgs& a;
    hipStream_t s;
    template <class T, int TPC, int NV> hipError_t go() { return launch_norm<T, TPC, NV>(a, s); }
};
struct NormGrad {
    const NormGradArgs& a;
    hipStream_t s;
    template <class T, int TPC, int NV> hipError_t go() { return launch_norm_grad<T, TPC, NV>(a, s); }
};
template <class F>
hipError_t by_type(int type, int n, F f) {
    return type == ELEM_F32 ? by_height<float>(n, f) : type == ELEM_F16 ? by_height<f16_t>(n, f) : by_height<bf16_t>(n, f);
}

}  // namespace

hipError_t rmsnorm(const NormArgs& all, hipStream_t s) {
    const long long size = (long long)elem_size(all.type), ng = all.group == 0 ? 1 : (all.nrows + all.group - 1) / all.group;
    for (long long c = 0; c < all.ncols; c += kSlabColumns) {
        NormArgs a = all;
        a.ncols = (int)(all.ncols - c < kSlabColumns ? all.ncols - c : kSlabColumns);
        a.X = (const char*)all.X + c * all.ldx * size;
        if (all.R) a.R = (const char*)all.R + c * all.ldr * size;
        if (all.H) a.H = (char*)all.H + c * all.ldh * size;
        if (all.Y) a.Y = (char*)all.Y + c * all.ldy * size;
        if (all.Q) {
            a.Q = all.Q + c * all.ldq;
            a.scales = all.scales + c * ng;
        }
        const hipError_t e = by_type(a.type, a.nrows, Norm{a, s});
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

hipError_t rmsnorm_grad(const NormGradArgs& all, hipStream_t s) {
    // columns of one launch: kNormMarks for every workgroup of the largest grid (256 threads and less, and 1024)
    const int n = all.nrows, slab = kNormMarks * (n <= 2048 ? norm_shares(256) : norm_shares(1024));
    const long long size = (long long)elem_size(all.type);
    for (long long c = 0; c < all.ncols; c += slab) {
        NormGradArgs a = all;
        a.ncols = (int)(all.ncols - c < slab ? all.ncols - c : slab);
        a.H = (const char*)all.H + c * all.ldh * size;
        a.dY = (const char*)all.dY + c * all.lddy * size;
        if (all.dH) a.dH = (const char*)all.dH + c * all.lddh * size;
        a.dX = (char*)all.dX + c * all.lddx * size;
        if (c > 0) a.beta = 1;
        NormGrad f{a, s};
        const hipError_t e = a.type == ELEM_F32 ? by_height_grad<float>(n, f) : a.type == ELEM_F16 ? by_height_grad<f16_t>(n, f) : by_height_grad<bf16_t>(n, f);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace bm
