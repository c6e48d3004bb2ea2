// C ABI of the operators over a model's columns (normalisation, routing, distillation, the 8-bit product): argument
// validation; the kernels are in rmsnorm.hip, route.hip, distill.hip and spmm_q8.hip.
#include "../../include/bidmat_hip.h"
#include "columns.hpp"
#include "common.hpp"
#include "elems.hpp"
#include "kernels.hpp"
#include "workspace.hpp"
#include <climits>
#include <initializer_list>
#include <cmath>

#define API extern "C" __attribute__((visibility("default")))

namespace {

constexpr int kInvalid = (int)hipErrorInvalidValue;

inline hipStream_t as_stream(void* s) { return reinterpret_cast<hipStream_t>(s); }

bool type_ok(int type) { return type == BIDMAT_F32 || type == BIDMAT_F16 || type == BIDMAT_BF16; }

// An operand of a call: a vector of n elements of `size` bytes, or a dense matrix of nrows x ncols with column stride ld.
struct Operand {
    const void* p;
    size_t size, n;
    long long rows, ld;      // ld 0: a vector
    bool out, aligned;
};
template <class T>
Operand vec(const T* p, long long n, bool out = false) {
    return {p, sizeof(T), (size_t)n, n, 0, out, (uintptr_t)p % sizeof(T) == 0};
}
Operand dense(const void* p, size_t size, int nrows, int ncols, long long ld, bool out = false) {
    return {p, size, (size_t)(ncols - 1) * (size_t)ld + nrows, nrows, ld, out, (uintptr_t)p % size == 0 && ld >= nrows};
}
// Whether two dense operands are different rows of one matrix: the same bytes from column to column, and no byte in common.
bool different_rows(const Operand& x, const Operand& y) {
    const size_t stride = (size_t)x.ld * x.size, wx = (size_t)x.rows * x.size, wy = (size_t)y.rows * y.size;
    if (x.ld == 0 || y.ld == 0 || stride != (size_t)y.ld * y.size) return false;
    const uintptr_t a = (uintptr_t)x.p, b = (uintptr_t)y.p;
    const size_t apart = (a < b ? b - a : a - b) % stride, from = a < b ? apart : (stride - apart) % stride;      // y's first byte behind x's
    return from >= wx && from + wy <= stride;
}
// Every operand given (p not null) lies at a multiple of its element, with columns apart; and no output shares memory with
// another operand, except a dense one that is a dense input, element by element.
bool operands_ok(std::initializer_list<Operand> all) {
    for (const Operand* x = all.begin(); x != all.end(); ++x) {
        if (!x->p) continue;
        if (!x->aligned) return false;
        for (const Operand* y = all.begin(); y != x; ++y) {
            if (!y->p || (!x->out && !y->out)) continue;
            const uintptr_t x0 = (uintptr_t)x->p, x1 = x0 + x->n * x->size, y0 = (uintptr_t)y->p, y1 = y0 + y->n * y->size;
            if (x0 >= y1 || y0 >= x1 || different_rows(*x, *y)) continue;
            const bool same = x->ld != 0 && x0 == y0 && x->ld == y->ld && x->size == y->size;
            if (!same || (x->out && y->out)) return false;
        }
    }
    return true;
}
bool group_ok(int group) { return group == 0 || group == 32 || group == 64 || group == 128; }

}  // namespace

API int bidmat_rmsnorm(int nrows, int ncols, int type, const void* X, int ldx, const void* R, int ldr, const float* w, float eps,
                       void* H, int ldh, void* Y, int ldy, unsigned char* Q, int ldq, float* scales, int group, void* stream) {
    if (nrows < 0 || ncols < 0 || !type_ok(type) || !group_ok(group) || !(eps >= 0.f) || std::isinf(eps)) return kInvalid;
    if (nrows > bm::kNormMaxRows || (Q == nullptr) != (scales == nullptr)) return kInvalid;
    if (nrows == 0 || ncols == 0) return 0;
    if (!X || !w || (!H && !Y && !Q)) return kInvalid;
    const size_t size = bm::elem_size(type);
    const long long ng = group == 0 ? 1 : (nrows + group - 1) / group;
    if (!operands_ok({dense(X, size, nrows, ncols, ldx), dense(R, size, nrows, ncols, ldr), vec(w, nrows), dense(H, size, nrows, ncols, ldh, true),
                      dense(Y, size, nrows, ncols, ldy, true), dense(Q, 1, nrows, ncols, ldq, true), vec(scales, ng * ncols, true)}))
        return kInvalid;
    bm::NormArgs a{nrows, ncols, type, X, R, ldx, ldr, w, eps, H, Y, ldh, ldy, Q, ldq, scales, group};
    return (int)bm::rmsnorm(a, as_stream(stream));
}

API int bidmat_rmsnorm_grad(int nrows, int ncols, int type, const void* H, int ldh, const float* w, float eps, const void* dY, int lddy,
                            const void* dH, int lddh, void* dX, int lddx, float* dw, int beta, void* stream) {
    auto lock = bm::device_lock();
    if (nrows < 0 || ncols < 0 || !type_ok(type) || !(eps >= 0.f) || std::isinf(eps) || (beta != 0 && beta != 1)) return kInvalid;
    if (nrows > bm::kNormMaxRows) return kInvalid;
    if (nrows == 0) return 0;
    if (ncols == 0) return dw && beta == 0 ? (int)bm::fill_f32(dw, nrows, 0.f, as_stream(stream)) : 0;
    if (!H || !w || !dY || !dX) return kInvalid;
    const size_t size = bm::elem_size(type);
    if (!operands_ok({dense(H, size, nrows, ncols, ldh), vec(w, nrows), dense(dY, size, nrows, ncols, lddy), dense(dH, size, nrows, ncols, lddh),
                      dense(dX, size, nrows, ncols, lddx, true), vec(dw, nrows, true)}))
        return kInvalid;
    bm::NormGradArgs a{nrows, ncols, type, H, dY, dH, ldh, lddy, lddh, w, eps, dX, lddx, dw, beta};
    return (int)bm::rmsnorm_grad(a, as_stream(stream));
}

API int bidmat_route(int nexperts, int ncols, int type, const void* Z, int ldz, const float* bias, int kind, int ngroups, int topgroups,
                     int topk, int renorm, float scale, float* Gdata, int* Gir, int* Gic, int* Gjc, int* counts, void* stream) {
    auto lock = bm::device_lock();
    if (nexperts < 1 || nexperts > bm::kRouteMaxExperts || ncols < 0 || !type_ok(type)) return kInvalid;
    if ((kind != BIDMAT_SOFTMAX && kind != BIDMAT_SIGMOID) || (renorm != 0 && renorm != 1)) return kInvalid;
    if (ngroups < 1 || ngroups > bm::kRouteMaxGroups || nexperts % ngroups != 0 || topgroups < 1 || topgroups > ngroups) return kInvalid;
    if (topk < 1 || topk > bm::kRouteMaxTop || topk > topgroups * (nexperts / ngroups)) return kInvalid;
    if (!std::isfinite(scale) || scale == 0.f || (long long)ncols * topk > INT_MAX) return kInvalid;
    if (ncols == 0) {
        hipError_t e = Gjc ? bm::fill_i32(Gjc, 1, 0, as_stream(stream)) : hipSuccess;
        if (e == hipSuccess && counts) e = bm::fill_i32(counts, nexperts, 0, as_stream(stream));
        return (int)e;
    }
    const long long nnz = (long long)ncols * topk;
    if (!Z || !Gdata || !Gir) return kInvalid;
    if (!operands_ok({dense(Z, bm::elem_size(type), nexperts, ncols, ldz), vec(bias, nexperts), vec(Gdata, nnz, true), vec(Gir, nnz, true),
                      vec(Gic, nnz, true), vec(Gjc, ncols + 1LL, true), vec(counts, nexperts, true)}))
        return kInvalid;
    bm::RouteArgs a{nexperts, ncols, type, Z, ldz, bias, kind, ngroups, topgroups, topk, renorm, scale, Gdata, Gir, Gic, Gjc, counts};
    return (int)bm::route(a, as_stream(stream));
}

API int bidmat_route_grad(int nexperts, int ncols, int type, const void* Z, int ldz, int kind, int topk, int renorm, float scale,
                          const float* Gdata, const int* Gir, const float* dG, void* dZ, int lddz, void* stream) {
    if (nexperts < 1 || nexperts > bm::kRouteMaxExperts || ncols < 0 || !type_ok(type)) return kInvalid;
    if ((kind != BIDMAT_SOFTMAX && kind != BIDMAT_SIGMOID) || (renorm != 0 && renorm != 1)) return kInvalid;
    if (topk < 1 || topk > bm::kRouteMaxTop || topk > nexperts || !std::isfinite(scale) || scale == 0.f) return kInvalid;
    if ((long long)ncols * topk > INT_MAX) return kInvalid;
    if (ncols == 0) return 0;
    if (!Z || !Gdata || !Gir || !dG || !dZ) return kInvalid;
    const long long nnz = (long long)ncols * topk;
    const size_t size = bm::elem_size(type);
    if (!operands_ok({dense(Z, size, nexperts, ncols, ldz), vec(Gdata, nnz), vec(Gir, nnz), vec(dG, nnz),
                      dense(dZ, size, nexperts, ncols, lddz, true)}))
        return kInvalid;
    bm::RouteGradArgs a{nexperts, ncols, type, Z, ldz, kind, topk, renorm, scale, Gdata, Gir, dG, dZ, lddz};
    return (int)bm::route_grad(a, as_stream(stream));
}

namespace {
int distill_call(const bm::DistillArgs& a, hipStream_t s) {
    if (a.nrows < 0 || a.nrows > (1 << 30) || a.ncols < 0 || !type_ok(a.type)) return kInvalid;
    if (a.nnz < 0 || a.nnz > INT_MAX - 1024) return kInvalid;          // the kernels count past a column's end, by a workgroup at most
    if (!(a.temperature >= 1e-18f) || !(a.temperature <= 1e18f)) return kInvalid;      // its square stays in the range of fp32
    if ((a.nrows == 0 || a.ncols == 0) && a.nnz > 0) return kInvalid;
    if (a.ncols == 0) return 0;
    if (a.nrows == 0) {
        // columns of nothing: loss 0, log-sum -inf
        if (!operands_ok({vec(a.loss, a.ncols, true), vec(a.lse, a.ncols, true)})) return kInvalid;
        hipError_t e = a.loss ? bm::fill_f32(a.loss, a.ncols, 0.f, s) : hipSuccess;
        if (e == hipSuccess && a.lse) e = bm::fill_f32(a.lse, a.ncols, -INFINITY, s);
        return e == hipErrorNoDevice ? 0 : (int)e;          // no device, no column: as with other calls that have no work
    }
    if (!a.Z || !a.tjc || (a.nnz > 0 && (!a.tdata || !a.tir))) return kInvalid;
    const size_t size = bm::elem_size(a.type);
    if (!operands_ok({dense(a.Z, size, a.nrows, a.ncols, a.ldz), vec(a.tdata, a.nnz), vec(a.tir, a.nnz), vec(a.tjc, a.ncols + 1LL),
                      vec(a.weight, a.ncols), vec(a.lse_in, a.ncols), vec(a.loss, a.ncols, true), vec(a.lse, a.ncols, true),
                      dense(a.dZ, size, a.nrows, a.ncols, a.lddz, true)}))
        return kInvalid;
    return (int)bm::distill(a, s);
}
}  // namespace

API int bidmat_distill(int nrows, int ncols, int type, const void* Z, int ldz, int nnz, const float* Tdata, const int* Tir, const int* Tjc,
                       float temperature, const float* weight, float* loss, float* lse, void* dZ, int lddz, void* stream) {
    auto lock = bm::device_lock();
    if (!loss && !lse && !dZ) return kInvalid;
    return distill_call({nrows, ncols, type, Z, ldz, nnz, Tdata, Tir, Tjc, temperature, weight, nullptr, loss, lse, dZ, lddz}, as_stream(stream));
}

API int bidmat_distill_grad(int nrows, int ncols, int type, const void* Z, int ldz, int nnz, const float* Tdata, const int* Tir,
                            const int* Tjc, float temperature, const float* weight, const float* lse, void* dZ, int lddz, void* stream) {
    auto lock = bm::device_lock();
    if (ncols > 0 && nrows > 0 && (!lse || !dZ)) return kInvalid;
    return distill_call({nrows, ncols, type, Z, ldz, nnz, Tdata, Tir, Tjc, temperature, weight, lse, nullptr, nullptr, dZ, lddz}, as_stream(stream));
}

API int bidmat_dsmult_q8_csc(int k, int ncols, int nnz, const unsigned char* Q, int ldq, const float* scales, int group, const float* Sdata,
                             const int* Sir, const int* Sjc, float* C, int beta, void* stream) {
    auto lock = bm::device_lock();
    if (k < 0 || k > (1 << 30) || ncols < 0 || nnz < 0 || !group_ok(group) || (beta != 0 && beta != 1)) return kInvalid;
    if (k == 0 || ncols == 0) return 0;
    if (ldq < k || !Sjc || !C || (nnz > 0 && (!Q || !scales || !Sdata || !Sir))) return kInvalid;
    // (the columns of A are not counted in the call: only its first one is known to be there)
    if (!operands_ok({dense(Q, 1, k, 1, ldq), vec(scales, 1), vec(Sdata, nnz), vec(Sir, nnz), vec(Sjc, ncols + 1LL),
                      dense(C, sizeof(float), k, ncols, k, true)}))
        return kInvalid;
    return (int)bm::dsmult_q8_csc(k, ncols, nnz, Q, ldq, scales, group, Sdata, Sir, Sjc, C, beta, as_stream(stream));
}
