// Distillation from a teacher's largest logits: the loss of a dense matrix of student logits Z (vocabulary x columns)
// against a sparse one of teacher logits T, and its gradient. With x = z / tau, t = T / tau, over one column:
//
//   p = softmax over the column's stored entries of t,   lse = log sum exp(x) over all rows
//   loss = weight * tau^2 * sum_j p_j (log p_j - x_{r_j} + lse),   dz_i = weight * tau * (exp(x_i - lse) - sum_{r_j = i} p_j)
//
// A column without stored entries, or with weight 0, has loss 0 and gradient 0, whatever its logits hold. A row may be
// stored twice; its shares add. Entries whose row lies outside the matrix are left out.
//
// What bounds it: memory. Loss and gradient of 131072 rows x 4096 columns in bf16: 430 us, 5.0 TB/s, every logit read once and
// written once; the gradient alone 355 us, 6.1 TB/s; the loss alone 253 us, 4.2 TB/s (128256 x 2048 fp32: 180 us, 5.9). Columns
// above 384 or 400 KiB (and above 128 KiB where there are few) are cut into chunks and read twice: 262144 x 512 fp32 299 us,
// 5.4 TB/s of what is moved; 128256 x 2048 fp32 584 us. Taking such columns in slabs that
// would stay in the 256 MB cache until the second time cost more than it gave (70000 x 2048 fp32: 344 us in slabs of 96 MiB, 399
// of 48, 324 in one). Few columns: two launches that leave no wait between them (100003 x 5 fp32: 3.9 and 5.0 us).
#include "columns.hpp"
#include "elems.hpp"
#include "kernels.hpp"
#include "workspace.hpp"

namespace bm {
namespace {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

// Columns in registers (k_distill_column) or cut into chunks (two launches): up to 128 KiB a column in one workgroup is
// faster however few there are (32768 bf16 rows: 8 columns 9.7 us against 12.7, 2048 columns 65 against 83); above, a
// workgroup of its own takes about 20 us, and below this many columns the chunks win (131072 bf16 rows: 64 columns 22 us
// against 17, 128 columns 24 against 22, 256 columns 33 against 45).
constexpr int kColumnsMin = 160;
// Columns of more than 256 KiB put their first vectors of eight into LDS, up to so many per thread (128 or 144 KiB): 1000 columns of
// 200064 bf16 rows 180 us, in chunks 238; 151936 rows 145 and 186; 70000 fp32 rows x 2048 columns 248 and 322. (A second round of
// the 256 CUs that is nearly empty costs some of it: 300 columns of 160000 rows 65 and 58.)
template <class T>
constexpr int kInLds = sizeof(T) == 2 ? 9 : 4;
// With the log-sums kept from an earlier call, columns of up to so many bytes (16384 columns bf16: 1000 rows 18 us against 38 by
// chunks, 2000 rows 35 against 50, 4000 rows 67 against 61).
constexpr size_t kKeptBytes = 6 << 10;
constexpr long long kSlabParts = 1 << 22;      // workgroups of one launch, at most

// Differences of logits are taken before they are scaled: a mask of the type's lowest value stays finite, and large
// common offsets cost no digits.
//
// What a column's teacher entries come to: p_j = exp((T_j - top) / tau - lsum). at0: the largest student logit among them,
// so that loss = tau^2 * weight * (part + mass * (lse - at0 / tau)) cancels nothing large.
struct Teacher {
    float top, lsum, part, mass, at0;
    int some, repeats;                   // whether an entry counts; whether a row is stored twice
};

// A running sum of 2^((z - top) * k), k = log2(e) / tau.
struct LogSum { float top, sum; };
__device__ __forceinline__ LogSum join(LogSum a, LogSum b, float k) {
    const float top = fmaxf(a.top, b.top);
    if (top == -INFINITY) return {top, a.sum + b.sum};          // both empty; a NaN in a sum stays
    return {top, a.sum * __builtin_amdgcn_exp2f((a.top - top) * k) + b.sum * __builtin_amdgcn_exp2f((b.top - top) * k)};
}
__device__ __forceinline__ LogSum wave_join(LogSum x, float k) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        LogSum y;
        y.top = __shfl_xor(x.top, m, 64);
        y.sum = __shfl_xor(x.sum, m, 64);
        x = join(x, y, k);
    }
    return x;
}
// All threads of a workgroup of 64 * waves get the joined log-sum.
__device__ __forceinline__ LogSum block_join(LogSum x, float k, LogSum* sh, int waves) {
    x = wave_join(x, k);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = x;
    __syncthreads();
    x = sh[0];
    for (int w = 1; w < waves; ++w) x = join(x, sh[w], k);
    return x;
}
// Eight more logits.
__device__ __forceinline__ LogSum add_eight(LogSum s, float8_t z, float k) {
    float top = s.top;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = fmaxf(top, z[j]);
    const float from = top == -INFINITY ? 0.f : top;
    float sum = s.sum * __builtin_amdgcn_exp2f((s.top - from) * k);
#pragma unroll
    for (int j = 0; j < 8; ++j) sum += __builtin_amdgcn_exp2f((z[j] - from) * k);
    return {top, sum};
}

// q = exp(z / tau - lse) = 2^((z + at * by) * k - off), from a column's log-sum or from a kept lse: the difference comes first,
// with one rounding. KEPT: never above 1. The lse of logits far from 0 has not the digits of log V, or (masks of the lowest
// value over a temperature below 1) is infinite, and 1 is what q cannot pass.
template <bool KEPT>
struct Share {
    float k, at, by, off;
    __device__ __forceinline__ float operator()(float z) const {
        const float e = fmaf(fmaf(at, by, z), k, -off);
        return __builtin_amdgcn_exp2f(KEPT ? __builtin_elementwise_minimum(e, 0.f) : e);          // a NaN stays one
    }
};
__device__ __forceinline__ Share<false> share_of(LogSum s, float k) { return {k, s.top, -1.f, __log2f(s.sum)}; }
__device__ __forceinline__ Share<true> share_of_lse(float lse, float tau, float k) { return {k, lse, -tau, 0.f}; }

__device__ __forceinline__ void column_entries(const DistillArgs& a, long long c, int& lo, int& hi) {
    lo = min(max(a.tjc[c], 0), a.nnz);
    hi = min(max(a.tjc[c + 1], lo), a.nnz);
}
__device__ __forceinline__ float column_scale(const DistillArgs& a, long long c) { return a.weight != nullptr ? a.weight[c] : 1.f; }

// One wave: whether a row is stored twice among n. Ascending rows show that they are not in one pass. Others set a bit each in
// a table in LDS. A few entries do so by a hash of the row, and one that finds its bit set is compared with the entries before
// it; with n^2 over four times the matrix's rows those comparisons would cost more than a pass over the entries for every
// 16384 rows, in which a bit is a row.
constexpr int kTableWords = 512, kTableBits = 32 * kTableWords;
__device__ int rows_repeat(const int* rows, int n, int nrows, unsigned* table) {
    const int lane = threadIdx.x & 63;
    bool ascend = true;
    for (int j = lane; j + 1 < n; j += 64) ascend = ascend && rows[j] < rows[j + 1];
    if (__ballot(!ascend) == 0) return 0;
    const bool hashed = (long long)n * n < 4LL * nrows;
    for (int base = 0, left = nrows; left > 0; base += kTableBits, left -= kTableBits) {
#pragma unroll
        for (int i = 0; i < kTableWords; i += 64) table[i + lane] = 0;
        for (int j0 = 0; j0 < n; j0 += 64) {
            const int r = j0 + lane < n ? rows[j0 + lane] : -1;
            const unsigned h = hashed ? ((unsigned)r * 2654435761u) >> 18 : (unsigned)r - (unsigned)base;
            const unsigned bit = 1u << (h & 31);
            const bool met = r >= 0 && h < kTableBits && (atomicOr(&table[h >> 5], bit) & bit) != 0;
            unsigned long long m = __ballot(met);
            if (!hashed && m != 0) return 1;
            for (; m != 0; m &= m - 1) {
                const int other = __builtin_amdgcn_readlane(r, __builtin_ctzll(m));
                int count = 0;
                for (int q = 0; q <= j0; q += 64) count += __popcll(__ballot(q + lane < n && rows[q + lane] == other));
                if (count > 1) return 1;
            }
        }
        if (hashed) return 0;
    }
    return 0;
}

// One wave: statistics of a column's teacher entries; at[] receives the student's logit at each of them. The first 64
// entries stay in registers, one per lane.
template <class T>
__device__ Teacher teacher_column(const DistillArgs& a, long long c, float it, float* at, unsigned* table) {
    const int lane = threadIdx.x & 63;
    int lo, hi;
    column_entries(a, c, lo, hi);
    const T* z = (const T*)a.Z + c * a.ldz;
    struct Entry { bool in; float t, z; };
    auto fetch = [&](int j) {
        const int r = a.tir[j];
        const float t = a.tdata[j];
        const bool in = (unsigned)r < (unsigned)a.nrows;
        return Entry{in, t, in ? (float)z[r] : 0.f};
    };
    Entry e0 = {false, 0.f, 0.f};
    if (lo + lane < hi) {
        e0 = fetch(lo + lane);
        at[lo + lane] = e0.z;
    }
    Teacher r;
    r.top = e0.in ? e0.t : -INFINITY;
    r.at0 = e0.in ? e0.z : -INFINITY;
    for (int j = lo + 64 + lane; j < hi; j += 64) {
        const Entry e = fetch(j);
        at[j] = e.z;
        if (e.in) {
            r.top = fmaxf(r.top, e.t);
            r.at0 = fmaxf(r.at0, e.z);
        }
    }
    r.top = group_allmax<64>(r.top);
    r.at0 = group_allmax<64>(r.at0);
    if (r.at0 == -INFINITY || r.at0 == INFINITY) r.at0 = 0.f;
    float sum = 0.f;
    bool some = false;
    auto add = [&](const Entry& e) {
        if (!e.in || e.t == -INFINITY) return;
        some = true;
        sum += expf((e.t - r.top) * it);
    };
    add(e0);
    for (int j = lo + 64 + lane; j < hi; j += 64) add(fetch(j));
    r.some = __ballot(some) != 0;
    r.lsum = logf(group_allsum<64>(sum));
    r.part = r.mass = 0.f;
    auto weigh = [&](const Entry& e) {
        const float logp = (e.t - r.top) * it - r.lsum, p = expf(logp);
        if (!e.in || p == 0.f) return;
        r.part += p * (logp - (e.z - r.at0) * it);
        r.mass += p;
    };
    weigh(e0);
    for (int j = lo + 64 + lane; j < hi; j += 64) weigh(fetch(j));
    r.part = group_allsum<64>(r.part);
    r.mass = group_allsum<64>(r.mass);
    r.repeats = rows_repeat(a.tir + lo, hi - lo, a.nrows, table);
    return r;
}

// Chunk `chunk` of column c: its log-sum (base 2). Workgroups behind the chunks take the teacher's columns, one wave each.
template <class T>
__global__ __launch_bounds__(BM_BLOCK) void k_distill_parts(DistillArgs a, int nchunks, int chunk, LogSum* parts, Teacher* stats, float* at) {
    __shared__ LogSum sh[BM_WAVES_PER_BLOCK];
    __shared__ unsigned table[BM_WAVES_PER_BLOCK][kTableWords];
    const float it = 1.f / a.temperature;
    const long long nparts = (long long)nchunks * a.ncols;
    if (blockIdx.x >= nparts) {
        const long long c = (blockIdx.x - nparts) * BM_WAVES_PER_BLOCK + (threadIdx.x >> 6);
        if (c >= a.ncols) return;
        const Teacher r = teacher_column<T>(a, c, it, at, table[threadIdx.x >> 6]);
        if ((threadIdx.x & 63) == 0) stats[c] = r;
        return;
    }
    const long long c = blockIdx.x / nchunks;
    const int b = (int)(blockIdx.x % nchunks);
    const T* z = (const T*)a.Z + c * a.ldz;
    const int lo = b * chunk, hi = min(a.nrows, lo + chunk);
    const float k = it * kLog2e;
    LogSum x = {-INFINITY, 0.f};
    for (int i = lo + (int)threadIdx.x * 8; i < hi; i += BM_BLOCK * 8) x = add_eight(x, load_col8(z, i, hi, (T)(-INFINITY)).wide(), k);
    x = block_join(x, k, sh, BM_WAVES_PER_BLOCK);
    if (threadIdx.x == 0) parts[blockIdx.x] = x;
}

__device__ __forceinline__ LogSum join_parts(const LogSum* parts, int nchunks, int t, int step, float k) {
    LogSum x = {-INFINITY, 0.f};
    for (int b = t; b < nchunks; b += step) x = join(x, parts[b], k);
    return x;
}

__device__ __forceinline__ void write_loss(const DistillArgs& a, long long c, LogSum s, float it, const Teacher& t) {
    const float l = __log2f(s.sum) * kLn2;
    if (a.lse != nullptr) a.lse[c] = fmaf(s.top, it, l);
    if (a.loss != nullptr) {
        const float w = column_scale(a, c);
        const float v = w * a.temperature * a.temperature * (t.part + t.mass * ((s.top - t.at0) * it + l));
        a.loss[c] = !t.some || w == 0.f ? 0.f : v;
    }
}

// Loss and log-sum alone: one wave per column.
__global__ __launch_bounds__(BM_BLOCK) void k_distill_loss(DistillArgs a, int nchunks, const LogSum* parts, const Teacher* stats) {
    const long long c = (long long)blockIdx.x * BM_WAVES_PER_BLOCK + (threadIdx.x >> 6);
    if (c >= a.ncols) return;
    const float it = 1.f / a.temperature, k = it * kLog2e;
    const LogSum x = wave_join(join_parts(parts + c * nchunks, nchunks, threadIdx.x & 63, 64, k), k);
    if ((threadIdx.x & 63) == 0) write_loss(a, c, x, it, stats[c]);
}

// The gradient at an entry of [e0, e1) in row r with the teacher's logit `value`, whose student logit was z, over its scale.
template <bool KEPT>
__device__ __forceinline__ float entry_grad(const DistillArgs& a, const Teacher& t, int e0, int e1, int r, float value, float z, float it,
                                            const Share<KEPT>& q) {
    float p = expf((value - t.top) * it - t.lsum);
    if (t.repeats) {
        p = 0.f;
        for (int i = e0; i < e1; ++i)
            if (a.tir[i] == r) p += expf((a.tdata[i] - t.top) * it - t.lsum);
    }
    return q(z) - p;
}

// The gradient of rows [lo, hi) of column c. ALONE: nothing was prepared and dZ is not Z: the log-sum is an earlier call's, and
// a fifth wave takes the teacher's entries while the others are at the column. Otherwise stats and at[] hold the
// teacher's statistics and the student's logits at its entries, parts the log-sums of the column's chunks (KEPT: lse_in has them).
template <class T, bool ALONE, bool KEPT>
__global__ __launch_bounds__(ALONE ? BM_BLOCK + 64 : BM_BLOCK) void k_distill_grad(DistillArgs a, int nchunks, int chunk, const LogSum* parts, const Teacher* stats,
                                                           const float* at) {
    __shared__ LogSum sh[BM_WAVES_PER_BLOCK];
    __shared__ Teacher own;
    __shared__ unsigned table[ALONE ? kTableWords : 1];
    constexpr int U = 4, STEP = BM_BLOCK * 8;            // loads in flight per thread
    const long long c = blockIdx.x / nchunks;
    const int b = (int)(blockIdx.x % nchunks), lo = b * chunk, hi = min(a.nrows, lo + chunk);
    const T* z = (const T*)a.Z + c * a.ldz;
    T* dz = (T*)a.dZ + c * a.lddz;
    int e0, e1;
    column_entries(a, c, e0, e1);
    const float w = column_scale(a, c) * a.temperature;
    const float lse = KEPT ? a.lse_in[c] : 0.f;
    bool none = e0 == e1 || w == 0.f;
    const bool extra = ALONE && threadIdx.x >= BM_BLOCK;
    const int i0 = extra ? hi : lo + (int)threadIdx.x * 8;
    Raw8<T> x[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (!none && i0 + u * STEP < hi) x[u] = load_col8(z, i0 + u * STEP, hi);
    const float it = 1.f / a.temperature;
    // the first entries are on their way while the column is
    const int j0 = e0 + (int)threadIdx.x;
    const bool early = !none && j0 < e1;
    const int r0 = early ? a.tir[j0] : -1;
    const float t0 = early ? a.tdata[j0] : 0.f, x0 = ALONE || !early ? 0.f : at[j0];
    const float k = it * kLog2e;
    Share<KEPT> q;
    Teacher t;
    if constexpr (ALONE) {
        q = share_of_lse(lse, a.temperature, k);
        if (extra && !none) {
            const int lane = threadIdx.x & 63;
            float sum = 0.f;
            bool some = false;
            t.top = -INFINITY;
            for (int j = e0 + lane; j < e1; j += 64)
                if ((unsigned)a.tir[j] < (unsigned)a.nrows) t.top = fmaxf(t.top, a.tdata[j]);
            t.top = group_allmax<64>(t.top);
            for (int j = e0 + lane; j < e1; j += 64)
                if ((unsigned)a.tir[j] < (unsigned)a.nrows && a.tdata[j] != -INFINITY) {
                    some = true;
                    sum += expf((a.tdata[j] - t.top) * it);
                }
            t.lsum = logf(group_allsum<64>(sum));
            t.some = __ballot(some) != 0;
            t.repeats = rows_repeat(a.tir + e0, e1 - e0, a.nrows, table);
            if (lane == 0) own = t;
        }
    } else {
        t = stats[c];
        if constexpr (KEPT) {
            q = share_of_lse(lse, a.temperature, k);
        } else {
            const LogSum s = block_join(join_parts(parts + c * nchunks, nchunks, threadIdx.x, BM_BLOCK, k), k, sh, BM_WAVES_PER_BLOCK);
            q = share_of(s, k);
            if (b == 0 && threadIdx.x == 0) write_loss(a, c, s, it, t);
        }
        none = none || !t.some;
    }
    auto rows = [&](auto part) {
#pragma unroll 1
        for (int i = i0; i < hi;) {
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (i + u * STEP < hi) {
                    float8_t v = (float8_t)(0.f);
                    if (!none) {
                        const float8_t y = x[u].wide();
#pragma unroll
                        for (int j = 0; j < 8; ++j) v[j] = part(y[j]);
                    }
                    store_col8(dz, i + u * STEP, hi, v);
                }
            i += U * STEP;
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (!none && i + u * STEP < hi) x[u] = load_col8(z, i + u * STEP, hi);
        }
    };
    if constexpr (KEPT) {
        // An lse of up to 2^16 is right to 2^-8, so that no q passes 1 by more, and its product with k is kept in two parts: the
        // first beside z * k with one rounding, the second (2^-24 of it) in the scale. That leaves a logit the instructions of an
        // exponential; the difference first, and the limit, cost two more (50001 x 2048 fp16: 85 us, so 84).
        const float base = q.at * a.temperature, most = base * k;
        const float wl = w * __builtin_amdgcn_exp2f(-fmaf(base, k, -most) - fmaf(q.at, a.temperature, -base) * k);
        const bool far = !none && !(fabsf(q.at) <= 0x1p16f);
        auto near_rows = [&] { rows([&](float v) { return wl * __builtin_amdgcn_exp2f(fmaf(v, k, -most)); }); };
        auto far_rows = [&] {
#pragma unroll 1
            for (int i = i0; i < hi; i += STEP) {
                float8_t v = load_col8(z, i, hi).wide();
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = w * q(v[j]);
                store_col8(dz, i, hi, v);
            }
        };
        if constexpr (ALONE) {          // dZ is not Z: a second pass, so that the first one stands by itself
            near_rows();
            if (far) far_rows();
        } else {
            if (far) far_rows();
            else near_rows();
        }
    } else {
        rows([&](float v) { return w * q(v); });
    }
    if (none) return;
    __syncthreads();          // the entries' values go over what other threads of the workgroup wrote
    if constexpr (ALONE) {
        t = own;
        if (!t.some) {          // entries, but none that counts
            for (int i = i0; i < hi; i += STEP) store_col8(dz, i, hi, (float8_t)(0.f));
            return;
        }
    }
    for (int j = j0; j < e1; j += (int)blockDim.x) {
        const int r = j == j0 ? r0 : a.tir[j];
        if (r < lo || r >= hi) continue;
        const float zr = ALONE ? (float)z[r] : j == j0 ? x0 : at[j];
        dz[r] = (T)(w * entry_grad(a, t, e0, e1, r, j == j0 ? t0 : a.tdata[j], zr, it, q));
    }
}

// A whole column in the registers of one workgroup of BLOCK threads, NV vectors of eight logits each: read once, written
// once; or the gradient alone, where log-sums are given. LV more vectors wait in LDS, each read back by the thread that put it
// there. The last wave takes the teacher's entries before its share of the column. Log-sums run along with the loads;
// afterwards the logits are still there as they were read.
// An entry's gradient goes over the one written for its row by the wave that wrote that one, whose stores take effect
// in order: no barrier has to wait for the column's stores.
template <class T, int BLOCK, int NV, int LV, bool KEPT>
__global__ __launch_bounds__(BLOCK) void k_distill_column(DistillArgs a, float* at) {
    constexpr int WAVES = BLOCK / 64;
    __shared__ LogSum sh[WAVES];
    __shared__ Teacher teacher;
    __shared__ unsigned table[kTableWords];
    __shared__ Raw8<T> kept_here[LV > 0 ? LV : 1][LV > 0 ? BLOCK : 1];
    const long long c = blockIdx.x;
    const int t = threadIdx.x, lane = t & 63, wave = wave_uniform(t >> 6), n = a.nrows;
    const float it = 1.f / a.temperature, k = it * kLog2e;
    const T* z = (const T*)a.Z + c * a.ldz;
    if (wave == WAVES - 1) {
        const Teacher r = teacher_column<T>(a, c, it, at, table);
        if (lane == 0) teacher = r;
    }
    Raw8<T> x[NV];
    LogSum s = {-INFINITY, 0.f};
    if constexpr (LV > 0) {
        Raw8<T> y[LV];
#pragma unroll
        for (int v = 0; v < LV; ++v) y[v] = load_col8(z, (v * BLOCK + t) * 8, n, (T)(-INFINITY));
#pragma unroll
        for (int v = 0; v < LV; ++v) {
            s = add_eight(s, y[v].wide(), k);
            kept_here[v][t] = y[v];
        }
        asm volatile("" : "+s"(z) : "v"(s.sum) : "memory");          // the rest is loaded when these registers are free
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) x[v] = load_col8(z, ((LV + v) * BLOCK + t) * 8, n, (T)(-INFINITY));
    if constexpr (KEPT) {
        __syncthreads();
    } else {
#pragma unroll
        for (int v = 0; v < NV; ++v) s = add_eight(s, x[v].wide(), k);
        s = block_join(s, k, sh, WAVES);
    }
    // 16-bit logits are widened again below: kept from above as floats they would take twice the registers
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int v = 0; v < NV; ++v) asm volatile("" : "+v"(x[v].v));
    }
    const Teacher tc = teacher;
    if (t == 0 && !KEPT) write_loss(a, c, s, it, tc);
    if (a.dZ == nullptr) return;
    T* dz = (T*)a.dZ + c * a.lddz;
    const float w = column_scale(a, c) * a.temperature;
    Share<KEPT> q;
    if constexpr (KEPT) q = share_of_lse(a.lse_in[c], a.temperature, k);
    else q = share_of(s, k);
    const bool none = !tc.some || w == 0.f;
    int e0, e1;
    column_entries(a, c, e0, e1);
    const bool first = !none && e0 + lane < e1;
    const int r0 = first ? a.tir[e0 + lane] : -1;
    const float x0 = first ? at[e0 + lane] : 0.f;
    int again = t;
    asm volatile("" : "+v"(again));          // read from LDS again, not kept in registers from above
    auto put = [&](const Raw8<T>& z8, int v) {
        float8_t d = (float8_t)(0.f);
        if (!none) {
            const float8_t y = z8.wide();
#pragma unroll
            for (int j = 0; j < 8; ++j) d[j] = w * q(y[j]);
        }
        store_col8(dz, (v * BLOCK + t) * 8, n, d);
    };
#pragma unroll
    for (int v = 0; v < LV; ++v) put(kept_here[v][again], v);
#pragma unroll
    for (int v = 0; v < NV; ++v) put(x[v], LV + v);
    if (none) return;
    for (int j = e0 + lane; j < e1; j += 64) {
        const int r = j < e0 + 64 ? r0 : a.tir[j];
        if ((unsigned)r >= (unsigned)n || ((r >> 3) & (BLOCK - 1)) >> 6 != wave) continue;
        dz[r] = (T)(w * entry_grad(a, tc, e0, e1, r, a.tdata[j], j < e0 + 64 ? x0 : at[j], it, q));
    }
}

template <class T, int BLOCK, int NV, int LV = 0>
hipError_t launch_column(const DistillArgs& a, float* at, hipStream_t s) {
    if constexpr (BLOCK == 64) {          // all that kKeptBytes lets through
        if (a.lse_in != nullptr) {
            hipLaunchKernelGGL((k_distill_column<T, BLOCK, NV, LV, true>), dim3((unsigned)a.ncols), dim3(BLOCK), 0, s, a, at);
            return hipGetLastError();
        }
    } else if (a.lse_in != nullptr) {
        return hipErrorInvalidValue;
    }
    hipLaunchKernelGGL((k_distill_column<T, BLOCK, NV, LV, false>), dim3((unsigned)a.ncols), dim3(BLOCK), 0, s, a, at);
    return hipGetLastError();
}
template <class T>
bool by_column(const DistillArgs& a) {
    const size_t bytes = sizeof(T) * (size_t)a.nrows;
    if (a.lse_in != nullptr) return bytes <= kKeptBytes;
    return bytes <= (128 << 10) || (bytes <= (256 << 10) + kInLds<T> * 1024 * 8 * sizeof(T) && a.ncols >= kColumnsMin);
}
template <class T>
hipError_t distill_columns(const DistillArgs& a, float* at, hipStream_t s) {
    const int vecs = (a.nrows + 7) / 8;
    // Small workgroups with as many vectors per thread as leave eight waves per SIMD: more columns at a time hide the way from
    // a column's pointer to its teacher's rows to the logits there (1000 rows x 16384 columns bf16: 25 us with one wave
    // per column, 49 with four; 20000 x 8192: 141 us with 512 threads, 212 with 1024). Larger columns take more registers.
    constexpr int M = sizeof(T) == 2 ? 8 : 4;
    if (vecs <= 64) return launch_column<T, 64, 1>(a, at, s);
    if (vecs <= 128) return launch_column<T, 64, 2>(a, at, s);
    if (vecs <= 64 * M / 2) return launch_column<T, 64, M / 2>(a, at, s);
    if (vecs <= 64 * M) return launch_column<T, 64, M>(a, at, s);
    if (vecs <= 128 * M * 3 / 4) return launch_column<T, 128, M * 3 / 4>(a, at, s);
    if (vecs <= 128 * M) return launch_column<T, 128, M>(a, at, s);
    if (vecs <= 256 * M * 3 / 4) return launch_column<T, 256, M * 3 / 4>(a, at, s);
    if (vecs <= 256 * M) return launch_column<T, 256, M>(a, at, s);
    if (vecs <= 512 * M * 3 / 4) return launch_column<T, 512, M * 3 / 4>(a, at, s);
    if (vecs <= 512 * M) return launch_column<T, 512, M>(a, at, s);
    if (vecs <= 768 * M) return launch_column<T, 512, M * 3 / 2>(a, at, s);
    if (vecs <= 1024 * M) return launch_column<T, 512, M * 2>(a, at, s);
    if (vecs <= 1536 * M) return launch_column<T, 1024, M * 3 / 2>(a, at, s);
    if (vecs <= 2048 * M) return launch_column<T, 1024, M * 2>(a, at, s);
    if constexpr (sizeof(T) == 2)
        if (vecs <= 1024 * (2 * M + 4)) return launch_column<T, 1024, M * 2, 4>(a, at, s);
    if (vecs <= 1024 * (2 * M + kInLds<T>)) return launch_column<T, 1024, M * 2, kInLds<T>>(a, at, s);
    return hipErrorInvalidValue;
}

template <class T>
hipError_t distill_typed(const DistillArgs& a, hipStream_t s) {
    // a chunk is a multiple of what a workgroup takes at once; smaller ones where there are few columns
    int chunk = 4 * BM_BLOCK * 8;
    while (chunk > BM_BLOCK * 8 && (long long)a.ncols * ((a.nrows + chunk - 1) / chunk) < 1024) chunk >>= 1;
    const int nchunks = (a.nrows + chunk - 1) / chunk;
    const long long nparts = (long long)nchunks * a.ncols;
    if (a.ncols > 1 && nparts + a.ncols > kSlabParts) {          // halves, until a launch holds them
        DistillArgs x = a, y = a;
        const long long half = a.ncols / 2, size = sizeof(T);
        x.ncols = (int)half;
        y.ncols = a.ncols - (int)half;
        y.Z = (const char*)a.Z + half * a.ldz * size;
        y.tjc += half;
        if (a.weight) y.weight += half;
        if (a.lse_in) y.lse_in += half;
        if (a.loss) y.loss += half;
        if (a.lse) y.lse += half;
        if (a.dZ) y.dZ = (char*)a.dZ + half * a.lddz * size;
        const hipError_t e = distill_typed<T>(x, s);
        return e != hipSuccess ? e : distill_typed<T>(y, s);
    }
    if (a.lse_in != nullptr && a.dZ != a.Z && !by_column<T>(a)) {
        hipLaunchKernelGGL((k_distill_grad<T, true, true>), dim3((unsigned)nparts), dim3(BM_BLOCK + 64), 0, s, a, nchunks, chunk, nullptr, nullptr, nullptr);
        return hipGetLastError();
    }
    hipError_t err;
    float* at = (float*)ws_get(WS_DISTILL_AT, sizeof(float) * (size_t)a.nnz, &err, s);
    if (!at) return err;
    if (by_column<T>(a)) return distill_columns<T>(a, at, s);
    char* buf = (char*)ws_get(WS_DISTILL, sizeof(Teacher) * (size_t)a.ncols + sizeof(LogSum) * (size_t)nparts, &err, s);
    if (!buf) return err;
    Teacher* stats = (Teacher*)buf;
    LogSum* parts = (LogSum*)(buf + sizeof(Teacher) * (size_t)a.ncols);
    const int waves = (a.ncols + BM_WAVES_PER_BLOCK - 1) / BM_WAVES_PER_BLOCK;
    const long long first = a.lse_in != nullptr ? waves : nparts + waves;
    hipLaunchKernelGGL((k_distill_parts<T>), dim3((unsigned)first), dim3(BM_BLOCK), 0, s, a, a.lse_in != nullptr ? 0 : nchunks, chunk, parts,
                       stats, at);
    if (a.dZ != nullptr)
        hipLaunchKernelGGL((a.lse_in != nullptr ? k_distill_grad<T, false, true> : k_distill_grad<T, false, false>), dim3((unsigned)nparts), dim3(BM_BLOCK), 0, s, a, nchunks, chunk, parts, stats, at);
    else
        hipLaunchKernelGGL(k_distill_loss, dim3((unsigned)waves), dim3(BM_BLOCK), 0, s, a, nchunks, parts, stats);
    return hipGetLastError();
}

}  // namespace

hipError_t distill(const DistillArgs& a, hipStream_t s) {
    return a.type == ELEM_F32 ? distill_typed<float>(a, s) : a.type == ELEM_F16 ? distill_typed<f16_t>(a, s) : distill_typed<bf16_t>(a, s);
}

}  // namespace bm
