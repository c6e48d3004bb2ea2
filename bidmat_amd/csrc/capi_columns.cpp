// C ABI of the operators over a model's columns (normalisation, routing, distillation, the 8-bit product): argument
// validation; the kernels are in rmsnorm.hip, route.hip, distill.hip and spmm_q8.hip.
#include "../../include/bidmat_hip.h"
#include "columns.hpp"
#include "common.hpp"
#include "elems.hpp"
#include "kernels.hpp"
#include "workspace.hpp"
#include <climits>
#include <cmath>

#define API extern "C" __attribute__((visibility("default")))

namespace {

constexpr int kInvalid = (int)hipErrorInvalidValue;

inline hipStream_t as_stream(void* s) { return reinterpret_cast<hipStream_t>(s); }

// A dense operand: nrows x ncols elements of `size` bytes, column stride ld.
struct Block {
    const void* p;
    long long ld;
    size_t size;
};
bool type_ok(int type) { return type == BIDMAT_F32 || type == BIDMAT_F16 || type == BIDMAT_BF16; }
bool block_ok(const Block& b, int nrows) { return b.ld >= nrows && (uintptr_t)b.p % b.size == 0; }
// Two operands of the same shape share memory in another way than element by element.
bool clash(const Block& x, const Block& y, int nrows, int ncols) {
    if (x.p == nullptr || y.p == nullptr) return false;
    if (x.p == y.p && x.ld == y.ld && x.size == y.size) return false;
    const uintptr_t x0 = (uintptr_t)x.p, x1 = x0 + ((size_t)(ncols - 1) * x.ld + nrows) * x.size;
    const uintptr_t y0 = (uintptr_t)y.p, y1 = y0 + ((size_t)(ncols - 1) * y.ld + nrows) * y.size;
    return x0 < y1 && y0 < x1;
}
// Two outputs share memory at all.
bool meet(const Block& x, const Block& y, int nrows, int ncols) {
    return x.p != nullptr && (x.p == y.p || clash(x, y, nrows, ncols));
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
    const Block in[2] = {{X, ldx, size}, {R, ldr, size}};
    const Block out[3] = {{H, ldh, size}, {Y, ldy, size}, {Q, ldq, 1}};
    for (const Block& b : in)
        if (b.p && !block_ok(b, nrows)) return kInvalid;
    for (int i = 0; i < 3; ++i) {
        if (!out[i].p) continue;
        if (!block_ok(out[i], nrows)) return kInvalid;
        for (const Block& b : in)
            if (clash(out[i], b, nrows, ncols)) return kInvalid;
        for (int j = 0; j < i; ++j)
            if (meet(out[i], out[j], nrows, ncols)) return kInvalid;
    }
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
    const Block in[3] = {{H, ldh, size}, {dY, lddy, size}, {dH, lddh, size}}, out = {dX, lddx, size};
    if (!block_ok(out, nrows)) return kInvalid;
    for (const Block& b : in)
        if (b.p && (!block_ok(b, nrows) || clash(out, b, nrows, ncols))) return kInvalid;
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
    if (!Z || !Gdata || !Gir || !block_ok({Z, ldz, bm::elem_size(type)}, nexperts)) return kInvalid;
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
    const Block z = {Z, ldz, bm::elem_size(type)}, dz = {dZ, lddz, bm::elem_size(type)};
    if (!block_ok(z, nexperts) || !block_ok(dz, nexperts) || clash(z, dz, nexperts, ncols)) return kInvalid;
    bm::RouteGradArgs a{nexperts, ncols, type, Z, ldz, kind, topk, renorm, scale, Gdata, Gir, dG, dZ, lddz};
    return (int)bm::route_grad(a, as_stream(stream));
}

namespace {
int distill_call(const bm::DistillArgs& a, hipStream_t s) {
    if (a.nrows < 0 || a.nrows > (1 << 30) || a.ncols < 0 || a.nnz < 0 || !type_ok(a.type)) return kInvalid;
    if (!(a.temperature > 0.f) || std::isinf(a.temperature) || std::isinf(1.f / a.temperature)) return kInvalid;
    if (a.nrows == 0 || a.ncols == 0) return a.nnz > 0 ? kInvalid : 0;
    if (!a.Z || !a.tjc || (a.nnz > 0 && (!a.tdata || !a.tir))) return kInvalid;
    const Block z = {a.Z, a.ldz, bm::elem_size(a.type)}, dz = {a.dZ, a.lddz, bm::elem_size(a.type)};
    if (!block_ok(z, a.nrows)) return kInvalid;
    if (a.dZ && (!block_ok(dz, a.nrows) || clash(z, dz, a.nrows, a.ncols))) return kInvalid;
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
    if (k < 0 || ncols < 0 || nnz < 0 || !group_ok(group) || (beta != 0 && beta != 1)) return kInvalid;
    if (k == 0 || ncols == 0) return 0;
    if (ldq < k || !Sjc || !C || (nnz > 0 && (!Q || !scales || !Sdata || !Sir))) return kInvalid;
    return (int)bm::dsmult_q8_csc(k, ncols, nnz, Q, ldq, scales, group, Sdata, Sir, Sjc, C, beta, as_stream(stream));
}
