// Int8 products grouped by expert (linear.hip).
#pragma once

#include "common.hpp"

namespace ohip {

struct LinearView {
    const int8_t* w;      // [experts][tiles][steps][1024]: 16 outputs x 64 inputs in lane order; gated: gate and up tiles alternate
    const float *scale, *bias;  // [experts][tiles * 16], bias null: none
    int experts, in, out;       // out: columns of the result
    int tiles, steps;
    int gated, act;
    float act_p0;
    int force;  // the launch that otter_hip_linear_set_kernel names, or -1
};
struct LinearRows {
    const float* x;
    size_t x_stride;
    int x_rows;
    const int32_t *index, *starts;  // null: the rows of x in their order, one expert
    int rows;
    float* y;
};
// Weights [experts][halves][out][in] into the tiles of LinearView (by the null stream).
hipError_t run_linear_pack(const int8_t* weight, int8_t* tiles, int experts, int out, int in, int halves);
size_t linear_workspace_bytes(const LinearView& w, int x_rows);
int linear_choice(const LinearView& w, int rows);  // otter_hip_linear_kernel_kind
size_t linear_groups(const LinearView& w, const LinearRows& r);  // workgroups of its launch
hipError_t run_linear(const LinearView& w, const LinearRows& r, void* workspace, hipStream_t stream);

}  // namespace ohip
