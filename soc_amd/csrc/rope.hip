// rope.hip - rotary positions of given rows (soc_rope_*): half or interleaved pairs, part of the head, scaled for long
// contexts, at positions in device memory. The reference's RopeOp (Mac/gpu/include/op/rope_op.h; soc_op_rope) rotates
// consecutive positions of unscaled half pairs in fp32.
#include <algorithm>
#include <cmath>
#include <memory>
#include <string>
#include <vector>

#include "capi_internal.h"
#include "rope.h"

namespace soc {
namespace {

// One row a block, or `parts` blocks where there are few rows. The first unit's values are requested before the angles are
// formed: cosines and sines (one double product, one sincospi a pair) serve all heads of the row from LDS.
// Bound by memory: 4093 rows x 16 heads of 128 fp16 values (33.5 MB) 8.2 us, 4.1 TB/s; 64 rows x 32 heads fp32 by the
// launch: 5.2 us a call, 3.0 of them the kernel's. One by one (pairs not in fours, or rows not 16-byte aligned) costs 1.5
// to 3 times that: 8000 rows x 40 heads of 80, 20 of them rotated, 48 us in fp32 and 46 in fp16, all 80 rotated 31 and 17.
template <typename T, int W>
__global__ __launch_bounds__(256) void k_rope_rows(RopeView v, const T* x, int64_t x_stride, T* y, int64_t y_stride,
                                                   int heads, const int32_t* __restrict__ positions, uint32_t offset,
                                                   int parts) {
  __shared__ f32x2 cs[kRopeMaxDim / 2];
  const int64_t r = blockIdx.x / parts;
  const int position = positions != nullptr ? positions[r] : static_cast<int>(offset + static_cast<uint32_t>(r));
  const int units = rope_units(v, W), all = heads * units;
  x += r * x_stride;
  y += r * y_stride;
  const int first = (blockIdx.x % parts) * 256 + threadIdx.x, step = parts * 256;
  const int early = min(first, all - 1);
  RopeUnit<T, W> unit = load_unit<T, W>(v, x + early / units * v.head_dim, early % units);
  rope_angles(v, position, cs);
  __syncthreads();
  for (int u = first; u < all; u += step) {
    if (u != first) unit = load_unit<T, W>(v, x + u / units * v.head_dim, u % units);
    store_unit<T, T, W>(v, cs, unit, y + u / units * v.head_dim, u % units);
  }
}

template <typename T>
hipError_t launch_rope_rows(const RopeView& v, const void* x, int64_t x_stride, void* y, int64_t y_stride, int rows,
                            int heads, const int32_t* positions, int offset, hipStream_t s) {
  constexpr int W = 16 / sizeof(T);
  const bool aligned = aligned_rows(x, x_stride, sizeof(T)) && aligned_rows(y, y_stride, sizeof(T));
  // 16 bytes a lane; 8 where pairs come in fours only; else element by element
  const int w = aligned && wide_units(v, W) ? W : aligned && wide_units(v, 4) ? 4 : 1;
  auto* k = w == W ? k_rope_rows<T, W> : w == 4 ? k_rope_rows<T, 4> : k_rope_rows<T, 1>;
  const int64_t units = static_cast<int64_t>(heads) * (v.rotary_dim / (2 * w) + (v.head_dim - v.rotary_dim) / w);
  const int parts = row_blocks(rows, units);
  for (int64_t r = 0; r < rows; r += kRowsALaunch) {
    const int n = static_cast<int>(std::min<int64_t>(kRowsALaunch, rows - r));
    hipLaunchKernelGGL(k, dim3(n * parts), dim3(256), 0, s, v, static_cast<const T*>(x) + r * x_stride, x_stride,
                       static_cast<T*>(y) + r * y_stride, y_stride, heads, positions != nullptr ? positions + r : nullptr,
                       static_cast<uint32_t>(offset) + static_cast<uint32_t>(r), parts);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

// Radians a position of each pair. The NTK base and the YaRN ramp follow the published methods (NTK-aware
// scaling; Peng et al., "YaRN", section 3).
std::vector<double> frequencies(const soc_rope_spec& c) {
  const int d = c.rotary_dim;
  const double theta =
      c.scaling == SOC_ROPE_NTK ? c.theta * std::pow(c.factor, static_cast<double>(d) / (d - 2)) : c.theta;
  std::vector<double> f(d / 2);
  for (int i = 0; i < d / 2; ++i) f[i] = std::pow(theta, -2.0 * i / d);
  if (c.scaling == SOC_ROPE_LINEAR)
    for (double& x : f) x /= c.factor;
  if (c.scaling == SOC_ROPE_YARN) {
    const double fast = c.beta_fast == 0 ? 32.0 : c.beta_fast, slow = c.beta_slow == 0 ? 1.0 : c.beta_slow;
    // the pair that turns `turns` times within the original length
    auto pair = [&](double turns) {
      return d * std::log(c.original_max_position / (turns * 2 * M_PI)) / (2 * std::log(theta));
    };
    const double low = std::max(0.0, std::floor(pair(fast))), high = std::min(d - 1.0, std::ceil(pair(slow)));
    const double width = high > low ? high - low : 0.001;
    for (int i = 0; i < d / 2; ++i) {
      const double ramp = std::min(1.0, std::max(0.0, (i - low) / width));
      f[i] = f[i] / c.factor * ramp + f[i] * (1 - ramp);
    }
  }
  return f;
}

int check_spec(const soc_rope_spec& c) {
  if (c.head_dim < 2 || c.head_dim > kRopeMaxDim || c.head_dim % 2 != 0)
    return fail(SOC_ERR_INVALID, "rope: head_dim must be even and 2 to 1024");
  if (c.rotary_dim < 2 || c.rotary_dim > c.head_dim || c.rotary_dim % 2 != 0)
    return fail(SOC_ERR_INVALID, "rope: rotary_dim must be even and 2 to head_dim");
  if (c.layout != SOC_ROPE_HALF && c.layout != SOC_ROPE_INTERLEAVED)
    return fail(SOC_ERR_INVALID, "rope: unknown pair layout");
  if (c.scaling < SOC_ROPE_UNSCALED || c.scaling > SOC_ROPE_YARN)
    return fail(SOC_ERR_INVALID, "rope: unknown scaling");
  if (!(c.theta > 1.0) || !std::isfinite(c.theta)) return fail(SOC_ERR_INVALID, "rope: theta must be above 1");
  if (c.scaling != SOC_ROPE_UNSCALED && (!(c.factor >= 1.0) || !std::isfinite(c.factor)))
    return fail(SOC_ERR_INVALID, "rope: factor must be at least 1");
  if (c.scaling == SOC_ROPE_NTK && c.rotary_dim <= 2)
    return fail(SOC_ERR_INVALID, "rope: NTK scaling needs rotary_dim above 2");
  if (c.scaling == SOC_ROPE_YARN) {
    if (c.original_max_position <= 0)
      return fail(SOC_ERR_INVALID, "rope: YaRN needs the original max position");
    if (!(c.beta_fast == 0 && c.beta_slow == 0) &&
        !(c.beta_slow > 0 && c.beta_fast > c.beta_slow && std::isfinite(c.beta_fast)))
      return fail(SOC_ERR_INVALID, "rope: YaRN needs beta_fast > beta_slow > 0, or both 0");
    if (!(c.attention_factor >= 0) || !std::isfinite(c.attention_factor))
      return fail(SOC_ERR_INVALID, "rope: attention_factor must not be negative");
  }
  return SOC_OK;
}

}  // namespace
}  // namespace soc

extern "C" {

int soc_rope_create(soc_ctx* ctx, const soc_rope_spec* spec, soc_rope** out) {
  SOC_API_BEGIN
  if (spec == nullptr || out == nullptr) return soc::fail(SOC_ERR_INVALID, "null argument");
  *out = nullptr;
  SOC_TRY(soc::check_spec(*spec));
  if (ctx == nullptr) return soc::fail(SOC_ERR_INVALID, "null context");
  soc::DeviceScope device(ctx);
  std::unique_ptr<soc_rope> r(new soc_rope());
  r->ctx = ctx;
  r->head_dim = spec->head_dim;
  r->rotary_dim = spec->rotary_dim;
  r->interleaved = spec->layout == SOC_ROPE_INTERLEAVED;
  if (spec->scaling == SOC_ROPE_YARN)
    r->gain = static_cast<float>(spec->attention_factor > 0 ? spec->attention_factor
                                                            : 0.1 * std::log(spec->factor) + 1);
  std::vector<double> f = soc::frequencies(*spec);
  for (double& x : f) x /= 2 * M_PI;
  hipError_t e = hipMalloc(&r->turns, f.size() * sizeof(double));
  if (e != hipSuccess) {
    (void)hipGetLastError();
    return soc::fail(SOC_ERR_NOMEM, "rope: allocation of the frequencies failed");
  }
  e = hipMemcpyAsync(r->turns, f.data(), f.size() * sizeof(double), hipMemcpyHostToDevice, ctx->stream);
  if (e == hipSuccess) e = hipStreamSynchronize(ctx->stream);
  if (e != hipSuccess) {
    (void)hipFree(r->turns);
    return soc::fail(SOC_ERR_HIP, std::string("rope: ") + hipGetErrorString(e));
  }
  *out = r.release();
  return SOC_OK;
  SOC_API_END
}

int soc_rope_destroy(soc_rope* rope) {
  SOC_API_BEGIN
  if (rope == nullptr) return SOC_OK;
  soc::DeviceScope device(rope->ctx);
  (void)hipStreamSynchronize(rope->ctx->stream);
  (void)hipFree(rope->turns);
  delete rope;
  return SOC_OK;
  SOC_API_END
}

int soc_rope_apply(const soc_rope* rope, const void* x, int64_t x_stride, void* y, int64_t y_stride, int32_t dtype,
                   int32_t rows, int32_t heads, const int32_t* positions, int32_t position_offset) {
  SOC_API_BEGIN
  if (dtype != SOC_DTYPE_F32 && dtype != SOC_DTYPE_F16) return soc::fail(SOC_ERR_INVALID, "rope: dtype must be F32 or F16");
  if (rows <= 0 || heads <= 0) return soc::fail(SOC_ERR_INVALID, "rope: need rows > 0 and heads > 0");
  if (x == y && x_stride != y_stride) return soc::fail(SOC_ERR_INVALID, "rope: in place needs equal strides");
  if (rope == nullptr) return soc::fail(SOC_ERR_INVALID, "null rope");
  const int64_t width = static_cast<int64_t>(heads) * rope->head_dim;
  if (width > (1 << 30)) return soc::fail(SOC_ERR_INVALID, "rope: rows of more than 2^30 elements");
  soc_ctx* ctx = rope->ctx;
  soc::DeviceScope device(ctx);
  soc::Operands operands(ctx);
  const int size = dtype == SOC_DTYPE_F32 ? 4 : 2;
  SOC_TRY(operands.rows("rope input", x, rows, x_stride, width, size));
  if (y != x) SOC_TRY(operands.rows("rope output", y, rows, y_stride, width, size));
  if (positions != nullptr) SOC_TRY(operands.array("rope positions", positions, rows, 4));
  const soc::RopeView v = soc::view_of(rope, rope->head_dim);
  const hipError_t e = size == 4 ? soc::launch_rope_rows<float>(v, x, x_stride, y, y_stride, rows, heads, positions,
                                                                position_offset, ctx->stream)
                                 : soc::launch_rope_rows<soc::f16>(v, x, x_stride, y, y_stride, rows, heads, positions,
                                                                   position_offset, ctx->stream);
  return e == hipSuccess ? SOC_OK : soc::fail(SOC_ERR_HIP, std::string("rope: ") + hipGetErrorString(e));
  SOC_API_END
}

}  // extern "C"
