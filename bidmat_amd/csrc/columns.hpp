// Host-side launchers of the operators over a model's columns (internal; capi_columns.cpp validates and calls these).
// `type` is an ElemType; leading dimensions count elements.
#pragma once
#include <hip/hip_runtime.h>

namespace bm {

constexpr int kNormMaxRows = 32768;      // a column lives in the registers of one workgroup
constexpr int kRouteMaxExperts = 1024;
constexpr int kRouteMaxTop = 64;
constexpr int kRouteMaxGroups = 64;

// A launch may not hold 2^32 threads: kernels with a grid over the columns take at most so many columns at once.
constexpr int kSlabColumns = 1 << 21;

struct NormArgs {
    int nrows, ncols, type;
    const void *X, *R;                   // R nullable
    long long ldx, ldr;
    const float* w;
    float eps;
    void *H, *Y;                         // nullable
    long long ldh, ldy;
    unsigned char* Q;                    // nullable, e4m3 codes
    long long ldq;
    float* scales;
    int group;                           // rows per scale: 0 (all), 32, 64, 128
};
hipError_t rmsnorm(const NormArgs& a, hipStream_t s);

struct NormGradArgs {
    int nrows, ncols, type;
    const void *H, *dY, *dH;             // dH nullable
    long long ldh, lddy, lddh;
    const float* w;
    float eps;
    void* dX;
    long long lddx;
    float* dw;                           // nullable
    int beta;
};
hipError_t rmsnorm_grad(const NormGradArgs& a, hipStream_t s);

struct RouteArgs {
    int nexperts, ncols, type;
    const void* Z;
    long long ldz;
    const float* bias;                   // nullable
    int kind, ngroups, topgroups, topk, renorm;
    float scale;
    float* data;
    int *ir, *ic, *jc, *counts;          // ic, jc, counts nullable
};
hipError_t route(const RouteArgs& a, hipStream_t s);

struct RouteGradArgs {
    int nexperts, ncols, type;
    const void* Z;
    long long ldz;
    int kind, topk, renorm;
    float scale;
    const float* data;
    const int* ir;
    const float* ddata;
    void* dZ;
    long long lddz;
};
hipError_t route_grad(const RouteGradArgs& a, hipStream_t s);

struct DistillArgs {
    int nrows, ncols, type;
    const void* Z;
    long long ldz;
    int nnz;
    const float* tdata;
    const int *tir, *tjc;
    float temperature;
    const float* weight;                 // nullable
    const float* lse_in;                 // nullable: log-sums kept from an earlier call
    float *loss, *lse;                   // nullable
    void* dZ;                            // nullable
    long long lddz;
};
hipError_t distill(const DistillArgs& a, hipStream_t s);

hipError_t dsmult_q8_csc(int k, int ncols, int nnz, const unsigned char* Q, long long ldq, const float* scales, int group,
                         const float* vals, const int* ir, const int* jc, float* C, int beta, hipStream_t s);

}  // namespace bm
