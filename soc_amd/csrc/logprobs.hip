// logprobs.hip - log probabilities of given tokens, their ranks, the entropy and the top alternatives of logit rows
// (soc_logprobs). The reference only samples from a row (Mac/gpu/src/runtime/sampler.cpp:14-71).
//
// With M the row's largest logit, d_i = (x_i - M) / temperature, S = sum exp(d_i) and D = sum d_i exp(d_i):
//   log p_i = d_i - log S,  entropy = log S - D / S.
// Differences are taken before they are scaled, so that nothing of the logits' common size enters the sums.
#include <cmath>
#include <string>

#include "capi_internal.h"
#include "device_common.h"

namespace soc {
namespace {

constexpr int kMaxTop = 64;

struct LogprobArgs {
  const void* logits;
  int64_t row_stride;
  int rows, vocab;
  float inv_t;  // 1 / temperature
  const int32_t* tokens;
  float* logprobs;
  int32_t* ranks;
  float* entropy;
  int top_n;
  int32_t* top_ids;
  float* top_logprobs;
};

// Order of logits as unsigned words: NaNs first, then by value, both zeros alike; never 0 nor all ones.
constexpr uint32_t kOrderNan = 0xffff0000u;  // above +inf's 0xff800000
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return kOrderNan;
  const uint32_t b = __float_as_uint(x + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t o) {
  if (o == kOrderNan) return __builtin_nanf("");
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
// Order of tokens: by logit, then by lowest id. Distinct for every token of a row; 0 is below all of them,
// all ones above.
__device__ __forceinline__ uint64_t key_of(float x, int id) {
  return static_cast<uint64_t>(order_of(x)) << 32 | static_cast<uint32_t>(~id);
}

// Running sums of a part of a row: largest logit, sum of exp(d), sum of d exp(d).
struct Sums {
  float m, s, d;
};
__device__ __forceinline__ Sums join(Sums a, Sums b, float inv_t) {
  const float m = fmaxf(a.m, b.m);
  if (m == -INFINITY) return Sums{m, 0.0f, 0.0f};
  Sums r{m, 0.0f, 0.0f};
  const float ua = (a.m - m) * inv_t, fa = expf(ua);  // a part of -inf alone has f = 0
  if (fa > 0.0f) {                                     // u may be -inf where f is 0
    r.s += a.s * fa;
    r.d += fa * (a.d + ua * a.s);
  }
  const float ub = (b.m - m) * inv_t, fb = expf(ub);
  if (fb > 0.0f) {
    r.s += b.s * fb;
    r.d += fb * (b.d + ub * b.s);
  }
  return r;
}

template <typename T>
__global__ __launch_bounds__(256) void k_logprobs(LogprobArgs a) {
  __shared__ Sums part[4];
  __shared__ uint64_t best[4];
  __shared__ int count[4];
  const int64_t r = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const T* x = static_cast<const T*>(a.logits) + r * a.row_stride;
  Sums u{-INFINITY, 0.0f, 0.0f};
  const int token = a.tokens != nullptr ? a.tokens[r] : -1;
  const bool given = token >= 0 && token < a.vocab;
  const uint64_t mine = given ? key_of(static_cast<float>(x[token]), token) : 0;
  int above = 0;
  bool bad = false;
  for (int i = tid; i < a.vocab; i += 256) {
    const float v = static_cast<float>(x[i]);
    bad |= !(v < INFINITY);
    above += key_of(v, i) > mine;
    u = join(u, Sums{v, v == -INFINITY ? 0.0f : 1.0f, 0.0f}, a.inv_t);
  }
  bad = __syncthreads_or(bad);
  for (int d = 1; d < 64; d <<= 1) {
    const Sums o{__shfl_xor(u.m, d), __shfl_xor(u.s, d), __shfl_xor(u.d, d)};
    u = join(u, o, a.inv_t);
    above += __shfl_xor(above, d);
  }
  if (lane == 0) {
    part[wid] = u;
    count[wid] = above;
  }
  __syncthreads();
  u = join(join(part[0], part[1], a.inv_t), join(part[2], part[3], a.inv_t), a.inv_t);
  above = count[0] + count[1] + count[2] + count[3];
  const float nan = __builtin_nanf("");
  const float log_s = u.s > 0.0f ? logf(u.s) : 0.0f;
  auto log_p = [&](float v) { return bad ? nan : v == -INFINITY ? -INFINITY : (v - u.m) * a.inv_t - log_s; };
  if (tid == 0) {
    if (a.tokens != nullptr) {
      a.logprobs[r] = given ? log_p(static_cast<float>(x[token])) : token == -1 ? 0.0f : nan;
      if (a.ranks != nullptr) a.ranks[r] = given ? above : -1;
    }
    if (a.entropy != nullptr) a.entropy[r] = bad ? nan : u.s > 0.0f ? log_s - u.d / u.s : 0.0f;
  }
  uint64_t below = ~0ull;
  for (int k = 0; k < a.top_n; ++k) {
    uint64_t w = 0;
    for (int i = tid; i < a.vocab; i += 256) {
      const uint64_t key = key_of(static_cast<float>(x[i]), i);
      if (key < below && key > w) w = key;
    }
    for (int d = 1; d < 64; d <<= 1) w = max(w, static_cast<uint64_t>(__shfl_xor(static_cast<unsigned long long>(w), d)));
    __syncthreads();
    if (lane == 0) best[wid] = w;
    __syncthreads();
    w = max(max(best[0], best[1]), max(best[2], best[3]));
    below = w;
    if (tid == 0) {
      a.top_ids[r * a.top_n + k] = static_cast<int32_t>(~static_cast<uint32_t>(w));
      a.top_logprobs[r * a.top_n + k] = log_p(value_of(static_cast<uint32_t>(w >> 32)));
    }
  }
}

}  // namespace
}  // namespace soc

extern "C" {

int soc_logprobs(soc_ctx* ctx, const void* logits, int32_t dtype, int64_t row_stride, int32_t rows, int32_t vocab,
                 float temperature, const int32_t* tokens, float* logprobs, int32_t* ranks, float* entropy,
                 int32_t top_n, int32_t* top_ids, float* top_logprobs) {
  SOC_API_BEGIN
  using soc::check_device_rows;
  if (dtype != SOC_DTYPE_F32 && dtype != SOC_DTYPE_F16)
    return soc::fail(SOC_ERR_INVALID, "logprobs: dtype must be F32 or F16");
  if (rows <= 0 || vocab <= 0 || vocab > (1 << 30))
    return soc::fail(SOC_ERR_INVALID, "logprobs: need rows > 0 and a vocabulary of 1 to 2^30");
  if (top_n < 0 || top_n > soc::kMaxTop || top_n > vocab)
    return soc::fail(SOC_ERR_INVALID, "logprobs: top_n must be 0 to min(64, vocab)");
  if (!std::isfinite(temperature) || (temperature > 0.0f && !std::isfinite(1.0f / temperature)))
    return soc::fail(SOC_ERR_INVALID, "logprobs: temperature and its inverse must be finite");
  if (tokens == nullptr && (logprobs != nullptr || ranks != nullptr))
    return soc::fail(SOC_ERR_INVALID, "logprobs: log probabilities and ranks need tokens");
  if (tokens == nullptr && entropy == nullptr && top_n == 0)
    return soc::fail(SOC_ERR_INVALID, "logprobs: nothing asked for");
  if (ctx == nullptr) return soc::fail(SOC_ERR_INVALID, "null context");
  soc::DeviceScope device(ctx);
  const int size = dtype == SOC_DTYPE_F32 ? 4 : 2;
  SOC_TRY(check_device_rows(ctx, "logprobs logits", logits, rows, row_stride, vocab, size));
  if (tokens != nullptr) {
    SOC_TRY(check_device_rows(ctx, "logprobs tokens", tokens, rows, 1, 1, 4));
    SOC_TRY(check_device_rows(ctx, "logprobs output", logprobs, rows, 1, 1, 4));
    if (ranks != nullptr) SOC_TRY(check_device_rows(ctx, "logprobs ranks", ranks, rows, 1, 1, 4));
  }
  if (entropy != nullptr) SOC_TRY(check_device_rows(ctx, "logprobs entropy", entropy, rows, 1, 1, 4));
  if (top_n > 0) {
    SOC_TRY(check_device_rows(ctx, "logprobs top_ids", top_ids, rows, top_n, top_n, 4));
    SOC_TRY(check_device_rows(ctx, "logprobs top_logprobs", top_logprobs, rows, top_n, top_n, 4));
  }
  soc::LogprobArgs a{logits, row_stride, rows,    vocab, temperature <= 0.0f ? 1.0f : 1.0f / temperature,
                     tokens, logprobs,   ranks,   entropy, top_n, top_ids, top_logprobs};
  auto* kernel = size == 4 ? soc::k_logprobs<float> : soc::k_logprobs<soc::f16>;
  hipLaunchKernelGGL(kernel, dim3(rows), dim3(256), 0, ctx->stream, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? SOC_OK : soc::fail(SOC_ERR_HIP, std::string("logprobs: ") + hipGetErrorString(e));
  SOC_API_END
}

}  // extern "C"
