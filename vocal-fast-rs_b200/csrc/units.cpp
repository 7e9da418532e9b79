// C ABI of the unit-head operators (declared in include/vfr_retrieval.h):
// argument checks, the device the pointers live on, workspace sizes.
#include "units.h"

#include <cmath>
#include <initializer_list>

#include "index_build.h"
#include "vfr_common.h"

namespace vfr {
namespace {

// Frames and units of the unit loss.  Its kernels hold tile coordinates in 32
// bits and look up to two tiles of 256 past the last row or unit.
constexpr int64_t kMaxUnitCount = int64_t(1) << 30;

// The device `p` lives on.  Kernels would fault on host memory, so it is
// refused; the other arguments are the caller's to keep on the same device.
int pointer_device(const void *p) {
    cudaPointerAttributes at{};
    cuda_check(cudaPointerGetAttributes(&at, p));
    require(at.type == cudaMemoryTypeDevice || at.type == cudaMemoryTypeManaged,
            "unit operator arguments must be device memory");
    return at.device;
}

int sm_count(int device) {
    int sms = 0;
    cuda_check(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
    return sms;
}

int current_sms() {
    int device = 0;
    cuda_check(cudaGetDevice(&device));
    return sm_count(device);
}

bool aligned_to(size_t bytes, std::initializer_list<const void *> pointers) {
    for (const void *p : pointers)
        if (reinterpret_cast<uintptr_t>(p) % bytes) return false;
    return true;
}

void check_rows(int64_t rows, int32_t width, int32_t dtype) {
    require(rows >= 0 && rows <= INT32_MAX, "row count must be in 0..2147483647");
    require(width >= 1 && width <= kMaxUnitWidth, "row width must be in 1..4096");
    require(dtype == kF32 || dtype == kBF16 || dtype == kF16, "unknown element type");
}

void check_units(int64_t rows, int32_t k, int32_t width, int32_t dtype) {
    check_rows(rows, width, dtype);
    require(dtype != kF16, "the unit loss takes f32 or bf16 frames (softmax gradients leave fp16's range)");
    require(k >= 1, "unit count must be positive");
    require(rows <= kMaxUnitCount && k <= kMaxUnitCount, "frames and units must number 2^30 at most");
}

cudaStream_t given_stream(const VfrStream *stream) {
    require(stream != nullptr, "null CUDA stream binding");
    return static_cast<cudaStream_t>(stream->stream);
}

}  // namespace
}  // namespace vfr

using vfr::cuda_check;
using vfr::guarded;
using vfr::require;

extern "C" int vfr_layer_norm(const void *x, const float *gamma, const float *beta, int64_t rows, int32_t width,
                              int32_t dtype, float eps, void *y, float *mean, float *rstd, uint8_t *packed,
                              uint8_t *exponents, VfrStream *stream, char **error) {
    return guarded(error, [&] {
        cudaStream_t s = vfr::given_stream(stream);
        vfr::check_rows(rows, width, dtype);
        require(std::isfinite(eps) && eps >= 0.0f, "layer norm eps must be finite and not negative");
        require(!packed == !exponents, "a checkpoint needs both its packed and its exponent buffer");
        if (rows == 0) return;
        require(x && y && mean && rstd, "null layer norm binding");
        require(vfr::aligned_to(vfr::dtype_bytes(dtype), {x, y}) && vfr::aligned_to(4, {gamma, beta, mean, rstd}),
                "misaligned layer norm binding");
        vfr::DeviceGuard guard(vfr::pointer_device(x));
        vfr::launch_layer_norm({x, gamma, beta, rows, width, dtype, eps, y, mean, rstd, packed, exponents},
                               vfr::current_sms(), s);
        cuda_check(cudaGetLastError());
    });
}

extern "C" int vfr_layer_norm_workspace(int64_t rows, int32_t width, size_t *bytes, char **error) {
    return guarded(error, [&] {
        require(bytes, "null workspace size output");
        vfr::check_rows(rows, width, vfr::kF32);
        *bytes = vfr::norm_backward_workspace(rows, width, vfr::current_sms());
    });
}

extern "C" int vfr_layer_norm_backward(const void *dy, const void *x, const uint8_t *packed,
                                       const uint8_t *exponents, const float *mean, const float *rstd,
                                       const float *gamma, int64_t rows, int32_t width, int32_t dtype, void *dx,
                                       float *dgamma, float *dbeta, void *workspace, size_t workspace_bytes,
                                       VfrStream *stream, char **error) {
    return guarded(error, [&] {
        cudaStream_t s = vfr::given_stream(stream);
        vfr::check_rows(rows, width, dtype);
        require(!packed == !exponents, "a checkpoint needs both its packed and its exponent buffer");
        require(!(x && packed), "layer norm gradients read the input or its checkpoint, not both");
        const bool params = dgamma || dbeta;
        if (rows == 0 && !params) return;
        require(rows == 0 || (dy && (x || packed) && mean && rstd && dx), "null layer norm binding");
        require(vfr::aligned_to(vfr::dtype_bytes(dtype), {dy, x, dx}) &&
                    vfr::aligned_to(4, {gamma, mean, rstd, dgamma, dbeta}) && vfr::aligned_to(16, {workspace}),
                "misaligned layer norm binding");
        vfr::DeviceGuard guard(vfr::pointer_device(rows > 0 ? dy : dgamma ? dgamma : dbeta));
        const int sms = vfr::current_sms();
        if (params && rows > 0)
            require(workspace && workspace_bytes >= vfr::norm_backward_workspace(rows, width, sms),
                    "layer norm workspace is too small");
        vfr::launch_layer_norm_backward({dy, x, packed, exponents, mean, rstd, gamma, rows, width, dtype, dx, dgamma,
                                         dbeta, static_cast<float *>(workspace)},
                                        sms, s);
        cuda_check(cudaGetLastError());
    });
}

extern "C" int vfr_checkpoint_pack(const void *x, int64_t rows, int32_t width, int32_t dtype, uint8_t *packed,
                                   uint8_t *exponents, VfrStream *stream, char **error) {
    return guarded(error, [&] {
        cudaStream_t s = vfr::given_stream(stream);
        vfr::check_rows(rows, width, dtype);
        if (rows == 0) return;
        require(x && packed && exponents, "null checkpoint binding");
        require(vfr::aligned_to(vfr::dtype_bytes(dtype), {x}), "misaligned checkpoint binding");
        vfr::DeviceGuard guard(vfr::pointer_device(x));
        vfr::launch_checkpoint_pack(x, rows, width, dtype, packed, exponents, vfr::current_sms(), s);
        cuda_check(cudaGetLastError());
    });
}

extern "C" int vfr_checkpoint_unpack(const uint8_t *packed, const uint8_t *exponents, int64_t rows, int32_t width,
                                     int32_t dtype, void *x, VfrStream *stream, char **error) {
    return guarded(error, [&] {
        cudaStream_t s = vfr::given_stream(stream);
        vfr::check_rows(rows, width, dtype);
        if (rows == 0) return;
        require(x && packed && exponents, "null checkpoint binding");
        require(vfr::aligned_to(vfr::dtype_bytes(dtype), {x}), "misaligned checkpoint binding");
        vfr::DeviceGuard guard(vfr::pointer_device(x));
        vfr::launch_checkpoint_unpack(packed, exponents, rows, width, dtype, x, vfr::current_sms(), s);
        cuda_check(cudaGetLastError());
    });
}

extern "C" int vfr_unit_loss_workspace(int64_t rows, int32_t k, int32_t width, int32_t dtype, int32_t backward,
                                       size_t *bytes, char **error) {
    return guarded(error, [&] {
        require(bytes, "null workspace size output");
        vfr::check_units(rows, k, width, dtype);
        *bytes = vfr::unit_loss_workspace(rows, k, width, dtype, backward != 0, vfr::current_sms());
    });
}

extern "C" int vfr_unit_loss(const void *x, const void *units, const float *bias, const int32_t *labels,
                             int64_t rows, int32_t k, int32_t width, int32_t dtype, float scale, float *loss,
                             float *lse, void *workspace, size_t workspace_bytes, VfrStream *stream, char **error) {
    return guarded(error, [&] {
        cudaStream_t s = vfr::given_stream(stream);
        vfr::check_units(rows, k, width, dtype);
        require(std::fabs(scale) <= 1e30f, "the logit scale must be finite (1e30 at most)");
        if (rows == 0) return;
        require(x && units && labels && loss && lse, "null unit loss binding");
        require(vfr::aligned_to(vfr::dtype_bytes(dtype), {x, units}) &&
                    vfr::aligned_to(4, {bias, labels, loss, lse}) && vfr::aligned_to(256, {workspace}),
                "misaligned unit loss binding");
        vfr::DeviceGuard guard(vfr::pointer_device(x));
        const int sms = vfr::current_sms();
        const size_t need = vfr::unit_loss_workspace(rows, k, width, dtype, false, sms);
        require(need == 0 || (workspace && workspace_bytes >= need), "unit loss workspace is too small");
        vfr::UnitLoss a{};
        a.x = x, a.units = units, a.bias = bias, a.labels = labels;
        a.rows = rows, a.k = k, a.width = width, a.dtype = dtype, a.scale = scale;
        a.loss = loss, a.lse = lse, a.workspace = workspace;
        vfr::launch_unit_loss(a, sms, s);
        cuda_check(cudaGetLastError());
    });
}

extern "C" int vfr_unit_loss_backward(const void *x, const void *units, const float *bias, const int32_t *labels,
                                      const float *lse, const float *dloss, int64_t rows, int32_t k, int32_t width,
                                      int32_t dtype, float scale, void *dx, void *dunits, float *dbias,
                                      void *workspace, size_t workspace_bytes, VfrStream *stream, char **error) {
    return guarded(error, [&] {
        cudaStream_t s = vfr::given_stream(stream);
        vfr::check_units(rows, k, width, dtype);
        require(std::fabs(scale) <= 1e30f, "the logit scale must be finite (1e30 at most)");
        require(units && dunits && (rows == 0 || (x && labels && lse && dloss && dx)), "null unit loss binding");
        require(vfr::aligned_to(vfr::dtype_bytes(dtype), {x, units, dx, dunits}) &&
                    vfr::aligned_to(4, {bias, labels, lse, dloss, dbias}) && vfr::aligned_to(256, {workspace}),
                "misaligned unit loss binding");
        vfr::DeviceGuard guard(vfr::pointer_device(units));
        const int sms = vfr::current_sms();
        if (rows == 0) {
            cuda_check(cudaMemsetAsync(dunits, 0, static_cast<size_t>(k) * width * vfr::dtype_bytes(dtype), s));
            if (dbias) cuda_check(cudaMemsetAsync(dbias, 0, static_cast<size_t>(k) * sizeof(float), s));
            return;
        }
        const size_t need = vfr::unit_loss_workspace(rows, k, width, dtype, true, sms);
        require(workspace && workspace_bytes >= need, "unit loss workspace is too small");
        vfr::UnitLoss a{};
        a.x = x, a.units = units, a.bias = bias, a.labels = labels;
        a.rows = rows, a.k = k, a.width = width, a.dtype = dtype, a.scale = scale;
        a.lse_in = lse, a.dloss = dloss, a.dx = dx, a.dunits = dunits, a.dbias = dbias, a.workspace = workspace;
        vfr::launch_unit_loss_backward(a, sms, s);
        cuda_check(cudaGetLastError());
    });
}
