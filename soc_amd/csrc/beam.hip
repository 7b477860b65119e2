// beam.hip - the best continuations of each request's beams over the vocabulary (soc_beam_select). The reference only samples
// from one row (Mac/gpu/src/runtime/sampler.cpp:14-71).
//
// score(b, v) = cum_b + (x_bv - M_b) / t - log S_b, with M_b the row's largest logit and S_b = sum exp((x_bv - M_b) / t).
// The terms of S are fp32 exponentials added in fp32 within a chunk; chunks are joined and scores formed in 64 bits: scores of a row
// are off by 5e-6 at most, all alike, so that they keep their order however near they are. A row's bits follow from its
// logits alone, not from where they lie: equal beams have equal scores.
#include <algorithm>
#include <cmath>
#include <string>

#include "paged_host.h"
#include "top_keys.h"

namespace soc {
namespace {

constexpr int kMaxStops = 8;
// Counters: each has a cache line to itself, where additions take their turns (64 requests of 8 beams, 19 chunks each: 71 us, with
// neighbouring counters 79).
constexpr int kApart = 32;

struct BeamRow {  // of a whole row: largest logit and log S; NaN where the row offers nothing
  double log_s;
  float m;
};
struct BeamArgs {
  const void* logits;
  int64_t row_stride;
  int beams, vocab;
  float to_log2;  // of a difference of logits
  double inv_t;
  const float* scores;
  int n;      // of each row's and of each group's first that are looked at
  int top_n;
  int stops[kMaxStops], num_stops;
  int chunks;  // of a row
  bool at_once;  // the last block of a request joins all chunks of its beams
  int first_row;                 // of the launch
  f32x2* parts;                  // [rows][chunks]: largest logit, sum
  uint64_t* tops;                // [rows][chunks][n]: first tokens in order, 0 where there are fewer
  BeamRow* rows;                 // [rows]
  uint64_t* row_tops;            // [rows][n]
  int *row_arrived, *group_arrived;  // zero between launches
  int32_t *top_rows, *top_tokens;
  float* top_scores;
  int32_t *next_rows, *next_tokens;
  float* next_scores;
};

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) v += __shfl_xor(v, d, kWave);
  return v;
}
template <typename T>
__device__ __forceinline__ void st_agent(T* p, T v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename T>
__device__ __forceinline__ T ld_agent(const T* p) {
  return __hip_atomic_load(const_cast<T*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// Whether this block is the last of `all` to come here; its earlier stores are seen by the last.
__device__ __forceinline__ bool arrives_last(int* arrived, int all, int* flag) {
  wait_mem();
  __syncthreads();
  if (threadIdx.x == 0) {
    *flag = atomicAdd(arrived, 1) == all - 1;
    if (*flag) st_dev(arrived, 0);
  }
  __syncthreads();
  return *flag != 0;
}
// Order of a score; 0 for none.
__device__ __forceinline__ uint64_t score_order(double s) {
  const uint64_t b = __builtin_bit_cast(uint64_t, s + 0.0);
  return b >> 63 ? ~b : b | uint64_t{1} << 63;
}
__device__ __forceinline__ double score_value(uint64_t o) {
  return __builtin_bit_cast(double, o >> 63 ? o & ~(uint64_t{1} << 63) : ~o);
}

// The n first tokens of a block's chunk, in order, to `first` (0 where it has fewer; a barrier before it is read), by all
// threads. A thread holds E logits v, logit e of id place(e) (of another thread: place_of(thread, e)), its largest `best`;
// ids outside [0, vocab) are no tokens and their logits -inf. keys: n * E words of LDS. Each thread's largest token stands
// for its E: the n-th largest of those keys is a threshold that at most n threads reach, so at most n E tokens (64 of
// normal data) are candidates, and those rank each other. No step here depends on how many values are equal. nans: whether a NaN
// may be among the logits. The rest is LDS; found and givers are 0 before the call, with a barrier since. (soc_logprobs has
// these steps in its kernel: calling this takes it 0.3 us of 11 for one row.)
template <typename T, int E, typename Place, typename PlaceOf>
__device__ __forceinline__ void block_first(const float (&v)[E], float best, bool nans, Place place, PlaceOf place_of,
                                            int vocab, int n, uint64_t* keys, uint64_t* first,
                                            uint64_t (&group)[kThreads], uint64_t& threshold, int (&giver)[kMaxTop],
                                            int& found, int& givers, int& tied) {
  constexpr int kLow = sizeof(T) == 2 ? 16 : 0;  // lowest bit of an order
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wid = tid / kWave;
  // the order of the thread's largest; 0 where it has no logit (the lowest of its ids is place(0), or 0). Where the sum
  // is NaN, a NaN may hide from `best`
  uint32_t order = place(0) < vocab ? order_of<T>(best) : 0;
  if (nans) {
    order = 0;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (place(e) >= 0 && place(e) < vocab) order = max(order, order_of<T>(v[e]));
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
        if ((v[e] == ov || (v[e] != v[e] && ov != ov)) && place(e) >= 0 && place(e) < vocab) id = place(e);
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
      if (id >= 0 && id < vocab && key >= t) keys[atomicAdd(&found, 1)] = key;
    }
  }
  __syncthreads();
  rank_first(keys, found, n, first);
}

// LDS beside the static: a chunk's candidates, or the first n of every chunk and those of them at the threshold; then the
// scores of every beam's first n, and which of them are at the threshold. At once: of every chunk's, and their keys.
__host__ __device__ constexpr size_t beam_room(int n, int each, int chunks, int beams, bool at_once) {
  const size_t row = static_cast<size_t>(n) * (at_once || each > 2 * chunks ? each : 2 * chunks) * 8;
  const size_t group = static_cast<size_t>(n) * beams * (at_once ? chunks * 20 : 12) + 8;
  return row > group ? row : group;
}
// Whether a request's chunks are joined at once, or row by row and then its rows. The second join takes 1 us (one request of 4
// beams, 151936 fp32 logits each, n 8: 12.9 us, at once 12.0), which the block that joins all makes up for where they have
// many first tokens (16 of 4 fp16 beams, n 12, 912 tokens a request: 19.4 us, at once 19.6). The threshold is sought among 256
// words, two or more a chunk.
constexpr bool joined_at_once(int n, int chunks, int beams) {
  return chunks > 1 && chunks * beams <= 128 && chunks * beams * n <= 768;
}

// One block per chunk of a row, as in soc_logprobs: 256 threads with E logits each in registers. The last block of a row to
// finish joins its chunks, the last of a request its beams; or that does both.
template <typename T, int E, bool kAtOnce>
__global__ __launch_bounds__(kThreads, E == 32 && sizeof(T) == 4 ? 8 : 4) void k_beam(BeamArgs a) {
  constexpr int VW = 16 / sizeof(T), NV = E / VW, C = kThreads * E;
  typedef T Vec __attribute__((ext_vector_type(VW), aligned(sizeof(T))));
  extern __shared__ uint64_t keys[];  // beam_room
  __shared__ uint64_t group[kThreads];
  __shared__ uint64_t first[kMaxTop];
  __shared__ float red[2][4];
  __shared__ uint64_t threshold;
  __shared__ int giver[kMaxTop];
  __shared__ int found, givers, flag, tied;
  __shared__ double row_log_s[kMaxTop];
  __shared__ float row_most[kMaxTop];

  const int64_t r = blockIdx.x / a.chunks;  // of the launch
  const int c = blockIdx.x % a.chunks, n = a.n;
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const T* x = static_cast<const T*>(a.logits) + (a.first_row + r) * a.row_stride;
  const int lo = c * C, base = lo + tid * VW;
  Vec raw[NV];
  if (lo + C <= a.vocab) {
#pragma unroll
    for (int k = 0; k < NV; ++k)
      raw[k] = __builtin_nontemporal_load(reinterpret_cast<const Vec*>(x + base + k * kThreads * VW));
  } else {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int i = base + k * kThreads * VW;
#pragma unroll
      for (int j = 0; j < VW; ++j) raw[k][j] = static_cast<T>(-INFINITY);
      if (i + VW <= a.vocab) {
        raw[k] = *reinterpret_cast<const Vec*>(x + i);
      } else {
#pragma unroll
        for (int j = 0; j < VW; ++j)
          if (i + j < a.vocab) raw[k][j] = x[i + j];
      }
    }
  }
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
  // -inf alone sums to 0; NaN, or +inf less itself, makes the sum NaN
  const float m0 = m == -INFINITY ? 0.0f : m;
  float part = 0.0f;
#pragma unroll
  for (int e = 0; e < E; ++e) part += __builtin_amdgcn_exp2f((v[e] - m0) * a.to_log2);
  part = wave_sum(part);
  if (lane == 0) red[1][wid] = part;
  __syncthreads();
  part = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
  block_first<T, E>(
      v, best, part != part, [&](int e) { return base + (e / VW) * kThreads * VW + e % VW; },
      [&](int thread, int e) { return lo + (thread + e / VW * kThreads) * VW + e % VW; }, a.vocab, n, keys, first, group,
      threshold, giver, found, givers, tied);
  __syncthreads();

  double s = part;
  // the wave's m and s of a whole row: lane l chunk l (at most 64)
  const auto whole = [&](int64_t row) {
    f32x2 mine = f32x2{-INFINITY, 0.0f};
    if (lane < a.chunks)
      mine = __builtin_bit_cast(f32x2, ld_agent(reinterpret_cast<const uint64_t*>(a.parts + row * a.chunks + lane)));
    m = wave_max(mine[0]);
    const double from = m == -INFINITY ? 0.0 : static_cast<double>(m);
    s = wave_sum(mine[1] * exp2((mine[0] - from) * (a.inv_t * 1.4426950408889634074)));
  };
  if (a.chunks > 1) {
    uint64_t* tops = a.tops + r * a.chunks * n;
    if (tid == 0) st_agent(reinterpret_cast<uint64_t*>(a.parts + r * a.chunks + c), __builtin_bit_cast(uint64_t, f32x2{m, part}));
    if (tid < n) st_agent(tops + c * n + tid, first[tid]);
  }
  if (!kAtOnce && a.chunks > 1) {
    const uint64_t* tops = a.tops + r * a.chunks * n;
    if (!arrives_last(a.row_arrived + r * kApart, a.chunks, &flag)) return;
    for (int i = tid; i < a.chunks * n; i += kThreads) keys[i] = ld_agent(tops + i);
    whole(r);  // by every wave
    // the first few of each chunk give a threshold that at least n of all keys reach, and seldom many more
    const int all = a.chunks * n, few = min(n, (n - 1) / a.chunks + 2);
    uint64_t* left = keys + all;
    if (tid == 0) found = 0;
    __syncthreads();
    if (wid == 0) {
      const auto key = [&](int i) { return keys[i / few * n + i % few]; };
      const uint64_t t = a.chunks * few <= kWave ? nth_largest<T, 1>(key, a.chunks * few, n)
                                                 : nth_largest<T, 4>(key, a.chunks * few, n);
      if (lane == 0) threshold = t;
    }
    if (tid < n) first[tid] = 0;
    __syncthreads();
    const uint64_t t = threshold;
    for (int i = tid; i < all; i += kThreads)
      if (keys[i] >= t) left[atomicAdd(&found, 1)] = keys[i];
    __syncthreads();
    rank_first(left, found, n, first);
    __syncthreads();
  }

  // the row, then the request's beams
  const int64_t g = r / a.beams;
  const auto log_of = [](double sum) {  // NaN: nothing but -inf, or a NaN or +inf among the logits
    return sum > 0.0 ? log(sum) : __builtin_nan("");
  };
  if (!kAtOnce) {
    if (tid < n) st_agent(a.row_tops + r * n + tid, first[tid]);
    if (tid == 0) {
      st_agent(reinterpret_cast<uint64_t*>(&a.rows[r].log_s), __builtin_bit_cast(uint64_t, log_of(s)));
      st_dev(&a.rows[r].m, m);
    }
  }
  const int lists = kAtOnce ? a.beams * a.chunks : a.beams, all = lists * n, per = all / a.beams;
  if (!arrives_last(a.group_arrived + g * kApart, lists, &flag)) return;
  const int row0 = static_cast<int>(g) * a.beams;  // of the launch
  const uint64_t* tops = (kAtOnce ? a.tops : a.row_tops) + static_cast<int64_t>(row0) * per;
  uint64_t* scores = keys;
  int* left = reinterpret_cast<int*>(keys + all);
  uint64_t* kept = keys + all + (all + 1) / 2;  // at once: the keys
  if (tid == 0) found = 0;
  if (kAtOnce) {
    for (int i = tid; i < all; i += kThreads) kept[i] = ld_agent(tops + i);
    for (int b = wid; b < a.beams; b += kThreads / kWave) {
      whole(row0 + b);
      if (lane == 0) {
        row_log_s[b] = log_of(s);
        row_most[b] = m;
      }
    }
    __syncthreads();
  }
  const auto key_of_place = [&](int i) { return kAtOnce ? kept[i] : ld_agent(tops + i); };
  for (int i = tid; i < all; i += kThreads) {
    const int b = i / per;
    const uint64_t key = key_of_place(i);
    const BeamRow* row = a.rows + row0 + b;
    const double log_sum = kAtOnce ? row_log_s[b]
                                   : __builtin_bit_cast(double, ld_agent(reinterpret_cast<const uint64_t*>(&row->log_s)));
    const float most = kAtOnce ? row_most[b] : ld_dev(&row->m), cum = a.scores[a.first_row + row0 + b];
    const float logit = value_of<T>(static_cast<uint32_t>(key >> 32));
    const double score = (static_cast<double>(logit) - most) * a.inv_t - log_sum + cum;
    // no token; a masked one; a beam that is none or whose row offers nothing
    scores[i] = key == 0 || !(score > -INFINITY) || !(score < INFINITY) ? 0 : score_order(score);
  }
  if (tid < n) group[tid] = ~uint64_t{0};
  __syncthreads();
  // candidates: all, or where they are many those at a threshold that at least n reach
  uint32_t t = 1;
  if (all > kThreads) {
    const int few = min(n, (n - 1) / lists + 2);  // at most 256 words
    if (wid == 0) {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = j * kWave + lane;
        w[j] = i < lists * few ? static_cast<uint32_t>(scores[i / few * n + i % few] >> 32) : 0;
      }
      bool exact;
      const uint32_t o = nth_word(w, n, 0, &exact);
      if (lane == 0) threshold = max(o, 1u);
    }
    __syncthreads();
    t = static_cast<uint32_t>(threshold);
  }
  for (int i = tid; i < all; i += kThreads)
    if (scores[i] >> 32 >= t) left[atomicAdd(&found, 1)] = i;
  __syncthreads();
  const int many = found;
  for (int k = tid; k < many; k += kThreads) {
    const int i = left[k];
    const uint64_t score = scores[i];
    int rank = 0, same = 0;
#pragma unroll 4
    for (int u = 0; u < many; ++u) {
      const uint64_t other = scores[left[u]];
      rank += other > score;
      same += other == score;
    }
    if (same > 1)  // the first beam's, then the larger logit's or the first token's
      for (int u = 0; u < many; ++u) {
        const int j = left[u];
        if (scores[j] == score) rank += kAtOnce && j / per == i / per ? kept[j] > kept[i] : j < i;
      }
    if (rank < n) group[rank] = i;
  }
  __syncthreads();
  if (wid != 0) return;
  int row = -1, token = -1;
  float score = -INFINITY;
  if (lane < n && group[lane] != ~uint64_t{0}) {
    const int i = static_cast<int>(group[lane]);
    row = a.first_row + row0 + i / per;
    token = kMaxVocab - static_cast<int32_t>(static_cast<uint32_t>(key_of_place(i)));
    score = static_cast<float>(score_value(scores[i]));
  }
  const int64_t request = a.first_row / a.beams + g;
  if (lane < a.top_n) {
    a.top_rows[request * a.top_n + lane] = row;
    a.top_tokens[request * a.top_n + lane] = token;
    a.top_scores[request * a.top_n + lane] = score;
  }
  if (a.next_rows == nullptr) return;
  bool goes_on = row >= 0;
  for (int k = 0; k < a.num_stops; ++k) goes_on &= token != a.stops[k];
  const uint64_t on = __ballot(goes_on);
  const int place = __popcll(on & ((uint64_t{1} << lane) - 1)), some = __popcll(on);
  const int64_t out = request * a.beams;
  if (goes_on && place < a.beams) {
    a.next_rows[out + place] = row;
    a.next_tokens[out + place] = token;
    a.next_scores[out + place] = score;
  }
  if (lane >= some && lane < a.beams) {
    a.next_rows[out + lane] = a.next_tokens[out + lane] = -1;
    a.next_scores[out + lane] = -INFINITY;
  }
}

template <typename T, int E>
hipError_t launch_beam(const BeamArgs& a, int rows, hipStream_t s) {
  hipLaunchKernelGGL((a.at_once ? k_beam<T, E, true> : k_beam<T, E, false>), dim3(static_cast<uint32_t>(rows) * a.chunks),
                     dim3(kThreads), beam_room(a.n, E, a.chunks, a.beams, a.at_once), s, a);
  return hipGetLastError();
}
template <typename T>
hipError_t launch_beam(const BeamArgs& a, int rows, int each, hipStream_t s) {
  return each == 32 ? launch_beam<T, 32>(a, rows, s) : launch_beam<T, 64>(a, rows, s);
}

}  // namespace
}  // namespace soc

extern "C" {

int soc_beam_select(soc_ctx* ctx, const void* logits, int32_t dtype, int64_t row_stride, int32_t groups, int32_t beams,
                    int32_t vocab, float temperature, const float* scores, const int32_t* stop_tokens, int32_t num_stops,
                    int32_t top_n, int32_t* top_rows, int32_t* top_tokens, float* top_scores, int32_t* next_rows,
                    int32_t* next_tokens, float* next_scores) {
  SOC_API_BEGIN
  if (dtype != SOC_DTYPE_F32 && dtype != SOC_DTYPE_F16)
    return soc::fail(SOC_ERR_INVALID, "beam select: dtype must be F32 or F16");
  if (groups <= 0 || beams <= 0 || beams > soc::kMaxTop || static_cast<int64_t>(groups) * beams > (1 << 20))
    return soc::fail(SOC_ERR_INVALID, "beam select: need groups > 0, 1 to 64 beams and at most 2^20 rows");
  if (vocab <= 0 || vocab > soc::kMaxVocab)
    return soc::fail(SOC_ERR_INVALID, "beam select: need a vocabulary of 1 to 2^20");
  if (!std::isfinite(temperature) || temperature > 0x1p100f || (temperature > 0.0f && !std::isfinite(2.0f / temperature)))
    return soc::fail(SOC_ERR_INVALID, "beam select: temperature must be at most 2^100, its inverse finite");
  const bool next = next_rows != nullptr || next_tokens != nullptr || next_scores != nullptr;
  if (num_stops < 0 || num_stops > soc::kMaxStops || (num_stops > 0 && stop_tokens == nullptr))
    return soc::fail(SOC_ERR_INVALID, "beam select: 0 to 8 stop tokens");
  if (top_n < 0 || top_n > soc::kMaxTop) return soc::fail(SOC_ERR_INVALID, "beam select: top_n must be 0 to 64");
  if (next && beams * (1 + num_stops) > soc::kMaxTop)
    return soc::fail(SOC_ERR_INVALID, "beam select: beams * (1 + stop tokens) must be at most 64");
  if (!next && top_n == 0) return soc::fail(SOC_ERR_INVALID, "beam select: nothing asked for");
  if (ctx == nullptr) return soc::fail(SOC_ERR_INVALID, "null context");
  soc::DeviceScope device(ctx);
  soc::Operands operands(ctx);
  const int size = dtype == SOC_DTYPE_F32 ? 4 : 2;
  const int64_t rows = static_cast<int64_t>(groups) * beams;
  SOC_TRY(operands.rows("beam select logits", logits, rows, row_stride, vocab, size));
  SOC_TRY(operands.array("beam select scores", scores, rows, 4));
  if (top_n > 0) {
    SOC_TRY(operands.rows("beam select top_rows", top_rows, groups, top_n, top_n, 4));
    SOC_TRY(operands.rows("beam select top_tokens", top_tokens, groups, top_n, top_n, 4));
    SOC_TRY(operands.rows("beam select top_scores", top_scores, groups, top_n, top_n, 4));
  }
  if (next) {
    SOC_TRY(operands.array("beam select next_rows", next_rows, rows, 4));
    SOC_TRY(operands.array("beam select next_tokens", next_tokens, rows, 4));
    SOC_TRY(operands.array("beam select next_scores", next_scores, rows, 4));
  }
  auto chunks_of = [&](int each) { return (vocab + soc::kThreads * each - 1) / (soc::kThreads * each); };
  // as in soc_logprobs: chunks of 8192 logits; of 16384 where a row is one of them then, and beyond 2^18
  const int each = (chunks_of(64) == 1 && chunks_of(32) > 1) || vocab > (1 << 18) ? 64 : 32;
  soc::BeamArgs a{};
  a.chunks = chunks_of(each);
  a.n = next ? std::max(top_n, beams * (1 + num_stops)) : top_n;
  a.at_once = soc::joined_at_once(a.n, a.chunks, beams);
  // groups a launch: its workspace stays below 32 MiB (or is one group's), its work-items below 2^32
  const size_t per_row = a.chunks * (8 + static_cast<size_t>(a.n) * 8) + sizeof(soc::BeamRow) + static_cast<size_t>(a.n) * 8 +
                         2 * soc::kApart * sizeof(int);
  const int64_t most = std::min<int64_t>((int64_t{32} << 20) / static_cast<int64_t>(per_row * beams),
                                         (int64_t{1} << 23) / (static_cast<int64_t>(a.chunks) * beams));
  const int step = static_cast<int>(std::min<int64_t>(groups, std::max<int64_t>(1, most)));
  const size_t step_rows = static_cast<size_t>(step) * beams;
  SOC_TRY(soc::ensure_serve_ws(ctx, step_rows * per_row, (step_rows + step) * soc::kApart));
  a.row_stride = row_stride;
  a.logits = logits;
  a.beams = beams;
  a.vocab = vocab;
  const double t = temperature <= 0.0f ? 1.0 : temperature;
  a.inv_t = 1.0 / t;
  a.to_log2 = static_cast<float>(1.4426950408889634074 / t);
  a.scores = scores;
  a.top_n = top_n;
  a.num_stops = next ? num_stops : 0;
  for (int k = 0; k < a.num_stops; ++k) a.stops[k] = stop_tokens[k];
  a.tops = reinterpret_cast<uint64_t*>(ctx->serve_ws);
  a.row_tops = a.tops + step_rows * a.chunks * a.n;
  a.rows = reinterpret_cast<soc::BeamRow*>(a.row_tops + step_rows * a.n);
  a.parts = reinterpret_cast<soc::f32x2*>(a.rows + step_rows);
  a.row_arrived = ctx->serve_counters;
  a.group_arrived = ctx->serve_counters + step_rows * soc::kApart;
  a.top_rows = top_rows;
  a.top_tokens = top_tokens;
  a.top_scores = top_scores;
  a.next_rows = next_rows;
  a.next_tokens = next_tokens;
  a.next_scores = next_scores;
  for (int32_t g = 0; g < groups; g += step) {
    a.first_row = g * beams;
    const int count = std::min(step, groups - g) * beams;
    const hipError_t e = size == 4 ? soc::launch_beam<float>(a, count, each, ctx->stream)
                                   : soc::launch_beam<soc::f16>(a, count, each, ctx->stream);
    if (e != hipSuccess) return soc::fail(SOC_ERR_HIP, std::string("beam select: ") + hipGetErrorString(e));
  }
  return SOC_OK;
  SOC_API_END
}

}  // extern "C"
