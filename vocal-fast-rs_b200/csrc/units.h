// Training a content encoder's unit head: layer norm and its gradients, 8-bit
// activation checkpoints (norm_kernels.cu, checkpoint_kernels.cu), and the
// softmax cross entropy of frames over a codebook of units with its gradients
// (unit_kernels.cu).  Argument checks are in units.cpp.
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace vfr {

enum { kF32 = 0, kBF16 = 1, kF16 = 2 };  // VFR_F32, VFR_BF16, VFR_F16
constexpr int kCheckpointBlock = 128;    // elements of a row that share one exponent
constexpr int kMaxUnitWidth = 4096;      // row width limit, as the retrieval index's

constexpr size_t dtype_bytes(int dtype) { return dtype == kF32 ? 4 : 2; }
constexpr int checkpoint_blocks(int width) { return (width + kCheckpointBlock - 1) / kCheckpointBlock; }

struct NormForward {
    const void *x;
    const float *gamma, *beta;  // either may be null (1, 0)
    int64_t rows;
    int width, dtype;
    float eps;
    void *y;
    float *mean, *rstd;
    uint8_t *packed, *exponents;  // both or neither
};
void launch_layer_norm(const NormForward &a, int sms, cudaStream_t stream);

struct NormBackward {
    const void *dy;
    const void *x;  // null: read packed / exponents instead
    const uint8_t *packed, *exponents;
    const float *mean, *rstd, *gamma;
    int64_t rows;
    int width, dtype;
    void *dx;
    float *dgamma, *dbeta;  // either may be null
    float *partials;        // norm_backward_workspace bytes
};
size_t norm_backward_workspace(int64_t rows, int width, int sms);
void launch_layer_norm_backward(const NormBackward &a, int sms, cudaStream_t stream);

void launch_checkpoint_pack(const void *x, int64_t rows, int width, int dtype, uint8_t *packed, uint8_t *exponents,
                            int sms, cudaStream_t stream);
void launch_checkpoint_unpack(const uint8_t *packed, const uint8_t *exponents, int64_t rows, int width, int dtype,
                              void *x, int sms, cudaStream_t stream);

struct UnitLoss {
    const void *x;      // [rows][width]
    const void *units;  // [k][width]
    const float *bias;  // [k] or null
    const int32_t *labels;
    int64_t rows;
    int k, width, dtype;
    float scale;
    // forward
    float *loss, *lse;
    // backward
    const float *lse_in, *dloss;
    void *dx, *dunits;
    float *dbias;  // null: not wanted
    void *workspace;
};
size_t unit_loss_workspace(int64_t rows, int k, int width, int dtype, bool backward, int sms);
void launch_unit_loss(const UnitLoss &a, int sms, cudaStream_t stream);
void launch_unit_loss_backward(const UnitLoss &a, int sms, cudaStream_t stream);

}  // namespace vfr
