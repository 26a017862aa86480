// Gradients with respect to the products of the linear layers (linear_grad.cu).
#pragma once

#include "linear.cuh"

namespace qsml {
namespace linear {

struct GradArgs {
    int64_t M = 0, N = 0;
    int act = QSML_ACT_NONE;
    const void* dy = nullptr;
    int64_t dy_ld = 0;
    const void* pre[2] = {nullptr, nullptr};  // rows of N; pre[0] null: dz = dy
    void* dz[2] = {nullptr, nullptr};         // rows of `pitch` (a multiple of 8), 16-byte aligned; null: not wanted
    int64_t pitch = 0;
    int64_t plane = 0;                        // > 0: dz in parts `plane` elements apart (Mat::plane)
    float* unscale = nullptr;                 // not null: a binary16 dz is stored times a power of two; 1 / it goes here
    ColumnSum db[2];
    float *partial = nullptr, *most = nullptr;  // workspace of the launch: column sums by part, the CTAs' largest |dz|,
    unsigned *arrived = nullptr, all = 0;       // the count of CTAs at the grid's barrier, and what it is when all are
    int* status = nullptr;
};

template <typename T> qsml_status_t run_grad(Context* ctx, const GradArgs& a, bool dual);

}  // namespace linear
}  // namespace qsml
