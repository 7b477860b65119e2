// logprobs.hip - log probabilities of given tokens, their ranks, the entropy and the top alternatives of logit rows
// (soc_logprobs). The reference only samples from a row (Mac/gpu/src/runtime/sampler.cpp:14-71).
//
// With M the row's largest logit, d_i = (x_i - M) / temperature, S = sum exp(d_i) and D = sum d_i exp(d_i):
//   log p_i = d_i - log S,  entropy = log S - D / S.
// Differences are taken before they are scaled, so that nothing of the logits' common size enters the sums. Two fp32
// logits can be further apart than fp32 reaches. A temperature above 1 could bring that back into its range, so from 1 on
// log p takes halves of the logits, subtracted in one fma, and twice the scale: the same bits otherwise. In the sums such
// a difference is -inf, whose exponential is the 0 that it has at temperatures up to 2^120 anyway (d below -256); beyond
// them the sums take halves too. Always taking them costs fp32 rows 2.5 % (777 x 151936 97.6 us for 95.2).
#include <algorithm>
#include <cmath>
#include <string>

#include "capi_internal.h"
#include "top_keys.h"

namespace soc {
namespace {

struct LogprobArgs {
  const void* logits;
  int64_t row_stride;
  int rows, vocab;
  float half;   // 1, or 1/2: what logits are multiplied by before they are subtracted
  float inv_t;  // 1 / (temperature * half)
  bool far;     // halves in the sums too
  const int32_t* tokens;
  float* logprobs;
  int32_t* ranks;
  float* entropy;
  int top_n;
  int32_t* top_ids;
  float* top_logprobs;
  int chunks;       // blocks a row
  struct Part* parts;    // [rows][chunks]
  uint64_t* tops;        // [rows][chunks][top_n]: each chunk's first tokens, 0 where it has fewer
  int* arrived;          // [rows], zero between launches
};

// One block per chunk of a row: 256 threads with E logits each in registers, read once in 16-byte loads, all requested
// before the first is used. The chunk's maximum comes first, so that every exponential is taken once; each thread counts
// its tokens before the given one, and one sum over the block follows. Of the top n, each thread's largest token stands
// for its E: the n-th largest of those 256 keys is a threshold that at most n threads reach, so at most n E tokens (64 of
// normal data) are candidates, and those rank each other. No step depends on how many values are equal. The last block of
// a row to finish joins its chunks, in chunk order.
// 777 rows of 151936 fp32 logits with top 8 take 96 us (4.9 TB/s; 87 us without alternatives, 5.4 TB/s). The same in fp16
// takes 87 us, so there the instructions a logit count, not memory. One row takes 10.7 us with top 20 and 5.3 without:
// the chain of reading, reducing, selecting, handing over and joining. At 32 fp32 logits a thread, 64 registers (8 waves
// a SIMD) are worth 5 % on many rows; in 16 bits they would spill.
// Keys in LDS: the candidates of a chunk (top_n threads of E tokens); then the top_n of every chunk that one block joins,
// and those of them at the threshold.
__host__ __device__ constexpr int key_room(int top_n, int each, int chunks) {
  return top_n * (each > 2 * chunks ? each : 2 * chunks);
}

struct Part {  // of a chunk: largest logit, sum of 2^d, sum of d 2^d (d: base-2 exponent below the largest), rank count
  float m, s, d;
  int above;
};

template <typename T, int E>
__global__ __launch_bounds__(kThreads, E == 32 && sizeof(T) == 4 ? 8 : 4) void k_logprobs(LogprobArgs a) {
  constexpr int VW = 16 / sizeof(T), NV = E / VW, C = kThreads * E;
  constexpr int kLow = sizeof(T) == 2 ? 16 : 0;  // lowest bit of an order
  typedef T Vec __attribute__((ext_vector_type(VW)));
  extern __shared__ uint64_t keys[];  // key_room(top_n, E, chunks)
  __shared__ uint64_t group[kThreads];
  __shared__ uint64_t first[kMaxTop];
  __shared__ float red[3][4];
  __shared__ int count[4];
  __shared__ uint64_t threshold;
  __shared__ int giver[kMaxTop];
  __shared__ int found, givers, last, tied;

  const int64_t r = blockIdx.x / a.chunks;
  const int c = blockIdx.x % a.chunks;
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const T* x = static_cast<const T*>(a.logits) + r * a.row_stride;
  // 16-byte loads start at the aligned address at or before the row, whose first logit is element `skip` of them
  const int skip = static_cast<int>(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T));
  const int base = c * C - skip + tid * VW;

  const int lo = c * C - skip, hi = lo + C;  // the chunk's ids, some of them outside the row at its ends
  const bool inner = lo >= 0 && hi <= a.vocab;
  // all loads are requested before any is used; what lies outside the row is -inf
  Vec raw[NV];
  if (inner) {
#pragma unroll
    for (int k = 0; k < NV; ++k)
      raw[k] = __builtin_nontemporal_load(reinterpret_cast<const Vec*>(x + base + k * kThreads * VW));
  } else {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int i = base + k * kThreads * VW;
#pragma unroll
      for (int j = 0; j < VW; ++j) raw[k][j] = static_cast<T>(-INFINITY);
      if (i >= 0 && i + VW <= a.vocab) raw[k] = *reinterpret_cast<const Vec*>(x + i);
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int i = base + k * kThreads * VW;
      if (i < a.vocab && i + VW > 0 && (i < 0 || i + VW > a.vocab)) {  // a vector across the row's first or last id
#pragma unroll
        for (int j = 0; j < VW; ++j)
          if (i + j >= 0 && i + j < a.vocab) raw[k][j] = x[i + j];
      }
    }
  }
  const int token = a.tokens != nullptr ? a.tokens[r] : -1;
  const bool given = token >= 0 && token < a.vocab;
  const float xt = given ? static_cast<float>(x[token]) : 0.0f;

  float v[E];
#pragma unroll
  for (int e = 0; e < E; ++e) v[e] = static_cast<float>(raw[e / VW][e % VW]);
  float best = v[0];
#pragma unroll
  for (int e = 1; e < E; ++e) best = fmaxf(best, v[e]);
  float m = wave_max(best);
  if (lane == 0) red[0][wid] = m;
  if (tid == 0) found = givers = 0;
  __syncthreads();
  m = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  // -inf alone sums to 0; NaN, or +inf less itself, makes the sums NaN
  const float m0 = m == -INFINITY ? 0.0f : m;
  const float to_log2 = a.inv_t * 1.4426950408889634f;  // of a difference of logits times `half`
  float s = 0.0f, d = 0.0f;
  auto add = [&](float u) {
    const float p = __builtin_amdgcn_exp2f(u);
    s += p;
    d = fmaf(p, fmaxf(u, -1000.0f), d);  // 2^-1000 is 0: a masked logit adds 0, not 0 times -inf
  };
  if (sizeof(T) == 4 && a.far) {
#pragma unroll
    for (int e = 0; e < E; ++e) add(fmaf(v[e], a.half, -m0 * a.half) * to_log2);
  } else {
    const float whole = to_log2 * a.half;
#pragma unroll
    for (int e = 0; e < E; ++e) add((v[e] - m0) * whole);
  }
  auto place_of = [&](int thread, int e) { return lo + (thread + e / VW * kThreads) * VW + e % VW; };
  auto place = [&](int e) { return base + (e / VW) * kThreads * VW + e % VW; };  // the id of the thread's logit e
  // tokens before the given one: equal logits at lower ids, larger ones anywhere. What is not of the row is -inf here,
  // which is never counted: ids below 0 are taken as large ones
  int above = 0;
  if (given) {
    if (xt != xt) {  // the NaNs before it: key by key, from the cache
      const uint64_t mine = key_of<T>(xt, token);
#pragma unroll 4
      for (int id = max(lo, 0) + tid; id < min(hi, a.vocab); id += kThreads)
        above += key_of<T>(static_cast<float>(x[id]), id) > mine;
    } else if (lo > token) {
#pragma unroll
      for (int e = 0; e < E; ++e) above += !(v[e] <= xt);
    } else if (lo >= 0 && hi <= token) {
#pragma unroll
      for (int e = 0; e < E; ++e) above += !(v[e] < xt);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        above += static_cast<uint32_t>(place(e)) < static_cast<uint32_t>(token) ? !(v[e] < xt) : !(v[e] <= xt);
    }
  }
  const float counts = wave_sum(static_cast<float>(above));  // exact: at most 2^20
  s = wave_sum(s);
  d = wave_sum(d);
  if (lane == 0) {
    red[1][wid] = s;
    red[2][wid] = d;
    count[wid] = static_cast<int>(counts);
  }
  __syncthreads();
  s = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
  d = (red[2][0] + red[2][1]) + (red[2][2] + red[2][3]);
  above = count[0] + count[1] + count[2] + count[3];

  const int n = a.top_n;
  if (n > 0) {
    // the order of the thread's largest; 0 where it has no logit (the lowest of its ids is place(0), or 0). Where the sum
    // is NaN, a NaN may hide from `best`
    uint32_t order = place(0) < a.vocab ? order_of<T>(best) : 0;
    if (s != s) {
      order = 0;
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (place(e) >= 0 && place(e) < a.vocab) order = max(order, order_of<T>(v[e]));
    }
    group[tid] = static_cast<uint64_t>(order) << 32;
    __syncthreads();
    uint32_t w[kThreads / kWave];  // wave 0
    if (wid == 0) {
#pragma unroll
      for (int j = 0; j < kThreads / kWave; ++j) w[j] = static_cast<uint32_t>(group[j * kWave + lane] >> 32);
      bool exact;
      const uint32_t o = nth_word(w, n, kLow, &exact);
      if (lane == 0) {
        threshold = static_cast<uint64_t>(o) << 32;
        tied = !exact && o != 0;
      }
    }
    __syncthreads();
    if (tied) {  // threads whose largest are equal at the threshold: those of the lowest ids
      const uint32_t o = static_cast<uint32_t>(threshold >> 32);
      if (order == o) {
        const float ov = value_of<T>(o);
        int id = 0;
#pragma unroll
        for (int e = E - 1; e >= 0; --e)
          if ((v[e] == ov || (v[e] != v[e] && ov != ov)) && place(e) >= 0 && place(e) < a.vocab) id = place(e);
        group[tid] |= low_of(id);
      }
      __syncthreads();
      if (wid == 0) {
        const int ties = n - reaching(w, o + 1);
#pragma unroll
        for (int j = 0; j < kThreads / kWave; ++j)
          w[j] = w[j] == o ? static_cast<uint32_t>(group[j * kWave + lane]) : 0;
        bool exact;
        const uint32_t low = nth_word(w, ties, 0, &exact);
        if (lane == 0) threshold |= low;
      }
    }
    if (tid < n) first[tid] = 0;
    __syncthreads();
    const uint64_t t = max(threshold, uint64_t{1});
    const float tv = value_of<T>(static_cast<uint32_t>(t >> 32));
    // the logits of the threads that reach it, at most n, are handed to all threads: E registers tested in place would be
    // E copies of what follows, mostly skipped (one row top 20 11.6 us for 10.7, 777 fp16 rows 91 for 87)
    float* handed = reinterpret_cast<float*>(keys);
    if (group[tid] >= t) {
      const int at = atomicAdd(&givers, 1);
      giver[at] = tid;
#pragma unroll
      for (int e = 0; e < E; ++e) handed[at * E + e] = v[e];
    }
    __syncthreads();
    const int all = __builtin_amdgcn_readfirstlane(givers * E);
    float y[kMaxTop * E / kThreads];
#pragma unroll
    for (int k = 0; k < kMaxTop * E / kThreads; ++k) {
      if (k * kThreads >= all) break;
      y[k] = handed[min(k * kThreads + tid, all - 1)];
    }
    __syncthreads();  // the keys take the logits' place
#pragma unroll
    for (int k = 0; k < kMaxTop * E / kThreads; ++k) {
      if (k * kThreads >= all) break;
      const int i = k * kThreads + tid;
      if (i < all && !(y[k] < tv)) {
        const int id = place_of(giver[i / E], i % E);
        const uint64_t key = key_of<T>(y[k], id);
        if (id >= 0 && id < a.vocab && key >= t) keys[atomicAdd(&found, 1)] = key;
      }
    }
    __syncthreads();
    rank_first(keys, found, n, first);
    __syncthreads();
  }

  if (a.chunks > 1) {
    Part* part = a.parts + r * a.chunks;
    uint64_t* tops = a.tops + r * a.chunks * n;
    if (tid == 0) {
      st_dev(&part[c].m, m);
      st_dev(&part[c].s, s);
      st_dev(&part[c].d, d);
      st_dev(&part[c].above, above);
    }
    if (tid < n)
      __hip_atomic_store(tops + c * n + tid, first[tid], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    wait_mem();
    __syncthreads();
    if (tid == 0) last = atomicAdd(a.arrived + r, 1) == a.chunks - 1;
    __syncthreads();
    if (!last) return;
    if (tid == 0) st_dev(a.arrived + r, 0);
    // every wave the same sums, lane l parts l and l + 64 (at most 65): requested with the keys
    Part mine[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int u = lane + j * kWave;
      mine[j] = Part{-INFINITY, 0.0f, 0.0f, 0};
      if (u < a.chunks) mine[j] = Part{ld_dev(&part[u].m), ld_dev(&part[u].s), ld_dev(&part[u].d), ld_dev(&part[u].above)};
    }
    for (int i = tid; i < a.chunks * n; i += kThreads)
      keys[i] = __hip_atomic_load(tops + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    m = wave_max(fmaxf(mine[0].m, mine[1].m));
    s = d = 0.0f;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const Part& p = mine[j];
      const float shift = p.m == -INFINITY ? -1000.0f : fmaxf(fmaf(p.m, a.half, -m * a.half) * to_log2, -1000.0f);
      const float f = __builtin_amdgcn_exp2f(shift);  // a NaN sum stays one: 0 times NaN is NaN
      s += p.s * f;
      d += f * (p.d + shift * p.s);
    }
    const float counted = static_cast<float>(mine[0].above + mine[1].above);  // exact: at most 2^20
    s = wave_sum(s);
    d = wave_sum(d);
    above = static_cast<int>(wave_sum(counted));
    if (n > 0) {
      // the first few of each chunk give a threshold that at least n of all keys reach, and seldom many more
      const int all = a.chunks * n, few = min(n, (n - 1) / a.chunks + 2);  // at most 64 + 2 * 65 words
      uint64_t* left = keys + all;
      __syncthreads();
      if (tid == 0) found = 0;
      if (wid == 0) {
        const auto key = [&](int i) { return keys[i / few * n + i % few]; };
        const uint64_t t = a.chunks * few <= kWave ? nth_largest<T, 1>(key, a.chunks * few, n)
                                                   : nth_largest<T, 4>(key, a.chunks * few, n);
        if (lane == 0) threshold = t;
      }
      __syncthreads();
      const uint64_t t = threshold;
      for (int i = tid; i < all; i += kThreads)
        if (keys[i] >= t) left[atomicAdd(&found, 1)] = keys[i];
      __syncthreads();
      rank_first(left, found, n, first);
      __syncthreads();
    }
  }

  const float nan = __builtin_nanf(""), ln2 = 0.6931471805599453f;
  const float log_s = s > 0.0f ? __builtin_amdgcn_logf(s) * ln2 : 0.0f;
  auto log_p = [&](float y) {
    return s != s ? nan : y == -INFINITY ? -INFINITY : fmaf(y, a.half, -m * a.half) * a.inv_t - log_s;
  };
  if (tid == 0) {
    if (a.tokens != nullptr) {
      a.logprobs[r] = given ? log_p(xt) : token == -1 ? 0.0f : nan;
      if (a.ranks != nullptr) a.ranks[r] = given ? above : -1;
    }
    if (a.entropy != nullptr) a.entropy[r] = s != s ? nan : s > 0.0f ? log_s - d / s * ln2 : 0.0f;
  }
  if (tid < n) {
    const uint64_t key = first[tid];
    a.top_ids[r * n + tid] = kMaxVocab - static_cast<int32_t>(static_cast<uint32_t>(key));
    a.top_logprobs[r * n + tid] = log_p(value_of<T>(static_cast<uint32_t>(key >> 32)));
  }
}

template <typename T, int E>
hipError_t launch_chunks(const LogprobArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((k_logprobs<T, E>), dim3(static_cast<uint32_t>(a.rows) * a.chunks), dim3(kThreads),
                     key_room(a.top_n, E, a.chunks) * sizeof(uint64_t), s, a);
  return hipGetLastError();
}
template <typename T>
hipError_t launch_logprobs(const LogprobArgs& a, int each, hipStream_t s) {
  return each == 32 ? launch_chunks<T, 32>(a, s) : launch_chunks<T, 64>(a, s);
}

}  // namespace
}  // namespace soc

extern "C" {

int soc_logprobs(soc_ctx* ctx, const void* logits, int32_t dtype, int64_t row_stride, int32_t rows, int32_t vocab,
                 float temperature, const int32_t* tokens, float* logprobs, int32_t* ranks, float* entropy,
                 int32_t top_n, int32_t* top_ids, float* top_logprobs) {
  SOC_API_BEGIN
  if (dtype != SOC_DTYPE_F32 && dtype != SOC_DTYPE_F16)
    return soc::fail(SOC_ERR_INVALID, "logprobs: dtype must be F32 or F16");
  if (rows <= 0 || vocab <= 0 || vocab > soc::kMaxVocab)
    return soc::fail(SOC_ERR_INVALID, "logprobs: need rows > 0 and a vocabulary of 1 to 2^20");
  if (top_n < 0 || top_n > soc::kMaxTop || top_n > vocab)
    return soc::fail(SOC_ERR_INVALID, "logprobs: top_n must be 0 to min(64, vocab)");
  if (!std::isfinite(temperature) || (temperature > 0.0f && !std::isfinite(2.0f / temperature)))
    return soc::fail(SOC_ERR_INVALID, "logprobs: temperature and its inverse must be finite");
  if (tokens == nullptr && (logprobs != nullptr || ranks != nullptr))
    return soc::fail(SOC_ERR_INVALID, "logprobs: log probabilities and ranks need tokens");
  if (tokens == nullptr && entropy == nullptr && top_n == 0)
    return soc::fail(SOC_ERR_INVALID, "logprobs: nothing asked for");
  if (ctx == nullptr) return soc::fail(SOC_ERR_INVALID, "null context");
  soc::DeviceScope device(ctx);
  soc::Operands operands(ctx);
  const int size = dtype == SOC_DTYPE_F32 ? 4 : 2;
  SOC_TRY(operands.rows("logprobs logits", logits, rows, row_stride, vocab, size));
  if (tokens != nullptr) {
    SOC_TRY(operands.array("logprobs tokens", tokens, rows, 4));
    SOC_TRY(operands.array("logprobs output", logprobs, rows, 4));
    if (ranks != nullptr) SOC_TRY(operands.array("logprobs ranks", ranks, rows, 4));
  }
  if (entropy != nullptr) SOC_TRY(operands.array("logprobs entropy", entropy, rows, 4));
  if (top_n > 0) {
    SOC_TRY(operands.rows("logprobs top_ids", top_ids, rows, top_n, top_n, 4));
    SOC_TRY(operands.rows("logprobs top_logprobs", top_logprobs, rows, top_n, top_n, 4));
  }
  const bool aligned = reinterpret_cast<uintptr_t>(logits) % 16 == 0 && row_stride * size % 16 == 0;
  const int skip = aligned ? 0 : 16 / size - 1;  // the most that a row's chunks start before it
  auto chunks_of = [&](int each) { return (vocab + skip + soc::kThreads * each - 1) / (soc::kThreads * each); };
  // chunks of 8192 logits (of 16384: 777 rows of 151936 top 8 102 us for 98, 64 in fp16 17.4 for 15.8); of 16384 where
  // a row is one of them then, without a join (200 rows of 16384 top 5 9.4 us for 11.9), and beyond 2^18, for fewer joins
  const int each = (chunks_of(64) == 1 && chunks_of(32) > 1) || vocab > (1 << 18) ? 64 : 32;
  const int chunks = chunks_of(each);
  const size_t per_row = chunks > 1 ? chunks * (sizeof(soc::Part) + static_cast<size_t>(top_n) * 8) : 0;
  // rows a launch: its workspace stays below 32 MiB, its work-items below 2^32
  const int64_t most = std::min<int64_t>(std::max<int64_t>(1, (int64_t{32} << 20) / std::max<size_t>(1, per_row)),
                                         (int64_t{1} << 23) / chunks);
  const int step = static_cast<int>(std::min<int64_t>(rows, most));
  if (chunks > 1) SOC_TRY(soc::ensure_serve_ws(ctx, step * per_row, step));
  soc::LogprobArgs a{};
  a.row_stride = row_stride;
  a.vocab = vocab;
  const float t = temperature <= 0.0f ? 1.0f : temperature;
  a.half = t >= 1.0f ? 0.5f : 1.0f;
  a.inv_t = 1.0f / (t * a.half);
  a.far = t > 0x1p120f;
  a.top_n = top_n;
  a.chunks = chunks;
  a.tops = reinterpret_cast<uint64_t*>(ctx->serve_ws);
  a.parts = reinterpret_cast<soc::Part*>(ctx->serve_ws + static_cast<size_t>(step) * chunks * top_n * 8);
  a.arrived = ctx->serve_counters;
  for (int64_t r = 0; r < rows; r += step) {
    a.logits = static_cast<const char*>(logits) + r * row_stride * size;
    a.rows = static_cast<int>(std::min<int64_t>(step, rows - r));
    a.tokens = tokens != nullptr ? tokens + r : nullptr;
    a.logprobs = logprobs != nullptr ? logprobs + r : nullptr;
    a.ranks = ranks != nullptr ? ranks + r : nullptr;
    a.entropy = entropy != nullptr ? entropy + r : nullptr;
    a.top_ids = top_n > 0 ? top_ids + r * top_n : nullptr;
    a.top_logprobs = top_n > 0 ? top_logprobs + r * top_n : nullptr;
    const hipError_t e = size == 4 ? soc::launch_logprobs<float>(a, each, ctx->stream)
                                   : soc::launch_logprobs<soc::f16>(a, each, ctx->stream);
    if (e != hipSuccess) return soc::fail(SOC_ERR_HIP, std::string("logprobs: ") + hipGetErrorString(e));
  }
  return SOC_OK;
  SOC_API_END
}

}  // extern "C"
