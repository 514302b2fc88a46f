// Beam search on slots: the selection of the next beams over beams and vocabulary, and the reordering of the slots they hold.
#include "common.cuh"

namespace mb200 {
namespace {

// ---- selection ------------------------------------------------------------------------------------------------------
// value[k,v] = score[k] + (logit[k,v] - logsumexp(logit[k])) of the B beams of a group; the `num` highest, ties to the lowest k V + v.
// Within a beam the order of the values is the order of the logits, so one pass over a beam's logits, cut into slices, gives
// each slice's maximum, its sum of exponentials and its `num` highest logits, and a second kernel, a CTA a group, joins them.
// A finished beam has one candidate, its end token at the beam's own score; a beam whose score is not finite, or whose logits hold a NaN, +inf or
// nothing above -inf, has none: what is no candidate counts as -inf, and still fills up places that are left, lowest first.
//
// The order is that of the values in 64 bits, at the price of 32: the logsumexp is off by a few 2^-20 (see too_close), and where candidates of
// different beams come that close, which is a few groups in a hundred calls, the joining CTA sums the group's exponentials again in 64 bits.

constexpr int kSelThreads = 256, kSelWarps = kSelThreads / 32, kSelPer = 32;             // logits of a thread
constexpr int kSelSlice = kSelThreads * kSelPer;
constexpr int kMostNum = 64, kMostBeams = 64;
constexpr int kList = 1024, kJoinList = 512;               // items side by side in shared memory

// By how much two logsumexps may be apart for rounding alone.  An exponent t = (v - top) log2(e) is off by 2.25 x 2^-24 |t| (a difference, a product,
// a constant), and the mean of |t| under the softmax is at most log2 of the vocabulary; ex2.approx is off by 2^-22 of its value; a thread
// adds 8 terms four times and those, and the threads' sums are added in 64 bits.  In units of 2^-24 of the sum, twice:
__device__ __forceinline__ double too_close(int V) { return 2 * 0x1p-24 * (2.25 * 0.6931472 * log2(double(V)) + 4. + 10.); }

// Unsigned order of floats, and of doubles.
__device__ __forceinline__ uint32_t order_of(float v) {
  const uint32_t u = __float_as_uint(v + 0.f);             // -0 and 0 are one value
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o); }
__device__ __forceinline__ uint64_t order_of(double v) {
  const uint64_t u = uint64_t(__double_as_longlong(v + 0.));
  return u >> 63 ? ~u : u | (uint64_t(1) << 63);
}
__device__ __forceinline__ double value_of(uint64_t o) {
  return __longlong_as_double(int64_t(o >> 63 ? o & ~(uint64_t(1) << 63) : ~o));
}
// An order and a place, the lower place ahead among equals.
__device__ __forceinline__ uint64_t key_of(float v, int place) { return uint64_t(order_of(v)) << 32 | uint32_t(~place); }

// A slice's part of a beam: its maximum and the sum of exp(logit - maximum) (NaN if it holds one).  Beside it, its highest logits
// as keys, highest first (0: no more).
struct Slice {
  float top, pad;
  double sum;
};

__device__ __forceinline__ uint64_t max64(uint64_t a, uint64_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint64_t min64u(uint64_t a, uint64_t b) { return a < b ? a : b; }

// The num-th highest of the lanes' keys (num <= 32): the lanes sort them.
__device__ __forceinline__ uint64_t nth_of_warp(uint64_t key, int num, int lane) {
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int step = size / 2; step >= 1; step >>= 1) {
      const uint64_t other = __shfl_xor_sync(0xffffffffu, key, step);
      const bool lower = (lane & step) == 0, falling = (lane & size) == 0;
      key = lower == falling ? max64(key, other) : min64u(key, other);
    }
  return __shfl_sync(0xffffffffu, key, num - 1);
}

// How the highest are found.  A warp in which num lanes hold a key as high as K holds num that high, so no key below K is wanted; K is the num-th
// highest of the lanes' own highest, and the CTA takes the highest K of its warps.  What reaches it (a few more than num in general) is put
// side by side and every item counts those ahead of it.  With more than 32 wanted the halves of a lane's logits stand for lanes, and K is
// the lowest of their 64.  Where more reach K than there is room for, num rounds of a maximum over the CTA find them.
// Bound: 8 instructions a logit (load and conversion, maximum, exponent, ex2, sum, two for the place of the maximum, one comparison with K), which
// is near the time that its 2 bytes take from HBM; three CTAs on an SM cover each other's barriers.
template <typename T, bool kVec>
__global__ void __launch_bounds__(kSelThreads, 3)
beam_slices_kernel(const T* __restrict__ logits, int64_t stride, int V, int num, Slice* __restrict__ slices, uint64_t* __restrict__ best) {
  __shared__ uint64_t s_list[kList], s_least[kSelWarps];
  __shared__ float s_top[kSelWarps];
  __shared__ double s_sum[kSelWarps];
  __shared__ int s_n;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t row = blockIdx.y, part = row * gridDim.x + blockIdx.x;
  const int v0 = int(blockIdx.x) * kSelSlice;
  const T* p = logits + row * stride;
  if (tid == 0) s_n = 0;
  cudaTriggerProgrammaticLaunchCompletion();               // the joining kernel may start, and waits for this one's end
  constexpr int kE = kVec ? Elem<T>::kVec : 1, kLoads = kSelPer / kE;
  float v[kSelPer];
  auto at = [&](int j) { return v0 + ((j / kE) * kSelThreads + tid) * kE + j % kE; };
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int c = at(i * kE);
    if (kVec && c + kE <= V) {
      if constexpr (kVec) {
        const Vec16<T> q = ldcs16(p + c);
#pragma unroll
        for (int k = 0; k < kE; ++k) v[i * kE + k] = Elem<T>::to_f(q.v[k]);
      }
    } else {
#pragma unroll
      for (int k = 0; k < kE; ++k) v[i * kE + k] = c + k < V ? Elem<T>::to_f(p[c + k]) : -INFINITY;
    }
  }
  // the highest of each half of the thread's logits, and where
  float high[2] = {-INFINITY, -INFINITY};
  int place[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int j = 0; j < kSelPer / 2; ++j) high[h] = fmaxf(high[h], v[h * kSelPer / 2 + j]);
    place[h] = at(h * kSelPer / 2);
#pragma unroll
    for (int j = kSelPer / 2 - 1; j >= 0; --j)
      if (v[h * kSelPer / 2 + j] == high[h]) place[h] = at(h * kSelPer / 2 + j);
  }
  float top = fmaxf(high[0], high[1]);
  const uint64_t key0 = key_of(high[0], place[0]), key1 = key_of(high[1], place[1]);
  uint64_t least;
  if (num <= 32) {
    least = nth_of_warp(max64(key0, key1), num, lane);
  } else {
    least = min64u(key0, key1);
#pragma unroll
    for (int s = 16; s >= 1; s >>= 1) least = min64u(least, __shfl_xor_sync(0xffffffffu, least, s));
  }
#pragma unroll
  for (int s = 16; s >= 1; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
  if (lane == 0) {
    s_top[warp] = top;
    s_least[warp] = least;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kSelWarps; ++w) {
    top = fmaxf(top, s_top[w]);
    least = max64(least, s_least[w]);
  }
  const float least_v = value_of(uint32_t(least >> 32));
  float sum4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < kSelPer; ++j) {
    sum4[j % 4] += ex2f((v[j] - top) * kLog2e);
    if (v[j] >= least_v) {
      const uint64_t key = key_of(v[j], at(j));
      if (key >= least && at(j) < V) {
        const int n = atomicAdd(&s_n, 1);
        if (n < kList) s_list[n] = key;
      }
    }
  }
  if (top == -INFINITY) {                                  // -inf - -inf: nothing to sum, unless there is a NaN
    sum4[0] = sum4[1] = sum4[2] = sum4[3] = 0.f;
#pragma unroll
    for (int j = 0; j < kSelPer; ++j)
      if (v[j] != v[j]) sum4[0] = v[j];
  }
  double all = (sum4[0] + sum4[1]) + (sum4[2] + sum4[3]);
#pragma unroll
  for (int s = 16; s >= 1; s >>= 1) all += __shfl_xor_sync(0xffffffffu, all, s);
  if (lane == 0) s_sum[warp] = all;
  __syncthreads();
  if (tid == 0) {
    all = 0.;
    for (int w = 0; w < kSelWarps; ++w) all += s_sum[w];
    slices[part] = Slice{top, 0.f, all};
  }
  const int n = s_n;
  uint64_t* const out = best + part * num;
  if (n <= kList) {
    for (int i = tid; i < n; i += kSelThreads) {
      const uint64_t key = s_list[i];
      int ahead = 0;
#pragma unroll 4
      for (int k = 0; k < n; ++k) ahead += s_list[k] > key;
      if (ahead < num) out[ahead] = key;
    }
    for (int i = n + tid; i < num; i += kSelThreads) out[i] = 0;
    return;
  }
  uint64_t last = ~uint64_t(0);
  for (int r = 0; r < num; ++r) {
    uint64_t key = 0;
#pragma unroll
    for (int j = 0; j < kSelPer; ++j) {
      const uint64_t k = key_of(v[j], at(j));
      if (at(j) < V && k < last) key = max64(key, k);
    }
#pragma unroll
    for (int s = 16; s >= 1; s >>= 1) key = max64(key, __shfl_xor_sync(0xffffffffu, key, s));
    __syncthreads();
    if (lane == 0) s_least[warp] = key;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kSelWarps; ++w) key = max64(key, s_least[w]);
    if (tid == 0) out[r] = key;
    last = key;
  }
}

// One CTA a group.  Candidates are looked at kSelThreads at a time; those ahead of the num-th highest so far go side by side in shared
// memory, and when there are many, and at the end, each counts those ahead of it.
__global__ void __launch_bounds__(kSelThreads)
beam_join_kernel(const Slice* __restrict__ slices, const uint64_t* __restrict__ best, const float* __restrict__ scores,
                 const uint8_t* __restrict__ finished, const void* __restrict__ logits, int64_t stride, int dtype, int beams, int n_slices, int V,
                 int num, int end_token, float* __restrict__ out_scores, int64_t* __restrict__ out_tokens, int64_t* __restrict__ out_parents) {
  __shared__ double s_total[kMostBeams];                   // logsumexp of a beam's logits less their maximum (which may be far beyond it)
  __shared__ float s_score[kMostBeams], s_top[kMostBeams];
  __shared__ uint8_t s_kind[kMostBeams];
  __shared__ double s_sum[kSelWarps];
  // an item: the value's order in 64 bits, and beam * V + token
  __shared__ uint64_t s_order[kJoinList + kMostNum];
  __shared__ uint64_t s_flat[kJoinList + kMostNum];
  __shared__ uint64_t s_best[2][kMostNum];
  __shared__ int s_n;
  enum { kOpen, kFinished, kDead };
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t g = blockIdx.x;
  cudaGridDependencySynchronize();
  for (int k = warp; k < beams; k += kSelWarps) {          // a warp a beam
    const int64_t row = g * beams + k;
    const Slice* const part = slices + row * n_slices;
    const float score = scores[row];
    int kind = kFinished;
    double total = 0.;
    float top = -INFINITY;
    if (!(finished && finished[row])) {
      for (int i = lane; i < n_slices; i += 32) top = fmaxf(top, part[i].top);
#pragma unroll
      for (int s = 16; s >= 1; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
      double sum = 0.;
      for (int i = lane; i < n_slices; i += 32) sum += part[i].sum * exp(double(part[i].top) - double(top));
#pragma unroll
      for (int s = 16; s >= 1; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
      kind = isfinite(top) && isfinite(sum) ? kOpen : kDead;
      if (kind == kOpen) total = log(sum);
    }
    if (lane == 0) {
      s_total[k] = total;
      s_score[k] = score;
      s_top[k] = top;
      s_kind[k] = uint8_t(isfinite(score) ? kind : kDead);
    }
  }
  __syncthreads();
  // Candidate i of the group: order (0: none) and place.  What is no candidate stands in at -inf, lowest tokens first: of those, a slice lists enough
  // among its highest logits if it has fewer than num others, and if one has not, no stand-in is needed.
  const int each = n_slices * num, all = beams * each;
  const uint64_t nothing = order_of(-double(INFINITY));
  auto candidate = [&](int i, uint64_t& flat) -> uint64_t {
    const int k = i / each, j = i - k * each, kind = s_kind[k];
    flat = uint64_t(k) * uint64_t(V);
    if (kind == kOpen) {
      const uint64_t key = best[g * all + i];
      flat += uint32_t(~uint32_t(key));
      return key ? order_of(double(s_score[k]) + ((double(value_of(uint32_t(key >> 32))) - double(s_top[k])) - s_total[k])) : 0;
    }
    if (kind == kFinished && j == 0) {
      flat += end_token;
      return order_of(double(s_score[k]));
    }
    int t = kind == kFinished ? j - 1 : j;
    if (kind == kFinished && t >= end_token) ++t;
    flat += t;
    return t < V && j < num ? nothing : 0;
  };
  for (bool again = false;; again = true) {
    uint64_t least_order = 0, least_flat = 0;              // of the num-th highest so far
    if (tid == 0) s_n = 0;
    __syncthreads();
    for (int base = 0; base < all; base += kSelThreads) {
      if (base + tid < all) {
        uint64_t flat;
        const uint64_t order = candidate(base + tid, flat);
        if (order && (order > least_order || (order == least_order && flat < least_flat))) {
          const int n = atomicAdd(&s_n, 1);
          s_order[n] = order;
          s_flat[n] = flat;
        }
      }
      __syncthreads();
      const int n = s_n;
      __syncthreads();
      if (n + kSelThreads <= kJoinList && base + kSelThreads < all) continue;
      for (int i = tid; i < n; i += kSelThreads) {
        const uint64_t order = s_order[i], flat = s_flat[i];
        int ahead = 0;
#pragma unroll 4
        for (int k = 0; k < n; ++k) {
          const uint64_t o = s_order[k];
          ahead += o > order || (o == order && s_flat[k] < flat);
        }
        if (ahead < num) {
          s_best[0][ahead] = order;
          s_best[1][ahead] = flat;
        }
      }
      __syncthreads();
      const int kept = min(n, num);
      if (tid < kept) {
        s_order[tid] = s_best[0][tid];
        s_flat[tid] = s_best[1][tid];
      }
      if (tid == 0) s_n = kept;
      if (kept == num) {
        least_order = s_best[0][num - 1];
        least_flat = s_best[1][num - 1];
      }
      __syncthreads();
    }
    if (again) break;
    // whether a candidate of another beam is too close to one that is chosen for 32 bits to tell them apart
    bool close = false;
    const double apart = too_close(V), edge = value_of(s_best[0][num - 1]) - apart;
    for (int i = tid; i < all && !close; i += kSelThreads) {
      uint64_t flat;
      const uint64_t order = candidate(i, flat);
      const double value = value_of(order);
      if (!order || !(value > -INFINITY) || value < edge) continue;
      const int k = i / each;
      for (int r = 0; r < num; ++r) {
        const double chosen = value_of(s_best[0][r]);
        if (fabs(chosen - value) > apart) continue;
        const int other = int(s_best[1][r] / uint64_t(V));
        close = close || (other != k && (s_kind[other] == kOpen || s_kind[k] == kOpen));
      }
    }
    if (!__syncthreads_or(close)) break;
    for (int k = 0; k < beams; ++k) {
      if (s_kind[k] != kOpen) continue;
      const int64_t from = (g * beams + k) * stride;
      const double top = s_top[k];
      double sum = 0.;
      for (int v = tid; v < V; v += kSelThreads) {
        const float x = dtype == MB200_F32 ? static_cast<const float*>(logits)[from + v]
                                           : __bfloat162float(static_cast<const __nv_bfloat16*>(logits)[from + v]);
        sum += exp(double(x) - top);
      }
#pragma unroll
      for (int s = 16; s >= 1; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
      __syncthreads();
      if (lane == 0) s_sum[warp] = sum;
      __syncthreads();
      if (tid == 0) {
        sum = 0.;
        for (int w = 0; w < kSelWarps; ++w) sum += s_sum[w];
        s_total[k] = log(sum);
      }
    }
    __syncthreads();
  }
  if (tid < num) {
    const uint64_t flat = s_best[1][tid];
    out_scores[g * num + tid] = float(value_of(s_best[0][tid]));
    out_parents[g * num + tid] = int64_t(flat / uint64_t(V));
    out_tokens[g * num + tid] = int64_t(flat % uint64_t(V));
  }
}

// ---- reordering -----------------------------------------------------------------------------------------------------
// new_slots[g,i] of the beam that goes on from beam parents[g,i]: the lowest child of a beam keeps its slot, the others take the slots of the
// beams without children, in order, and get copies.  Nothing that is copied from is written, so all copies run at once, in place: of every
// pool, and only those that a beam with several children makes necessary.  A parent that is no beam is nobody: its child takes a slot
// like a further child, and nothing is copied.
//
// Every CTA makes the list of copies for itself in shared memory (a launch and a round trip through global memory less), then takes its share of
// (copy, part of a state) pairs.  Bound by HBM: each copied byte is read and written once.
constexpr int kReorderThreads = 256, kReorderPart = 16384;  // bytes a CTA copies at a time
constexpr int kMostSlotBeams = 4096, kMostPools = 128;

struct Pools {
  char* at[kMostPools];
  int64_t bytes[kMostPools];                               // of an entry
  int first_part[kMostPools + 1];                          // parts of an entry in the pools in front
  int n;
};

template <int kBytes> struct Word;
template <> struct Word<16> { using type = uint4; };
template <> struct Word<4> { using type = uint32_t; };
template <> struct Word<1> { using type = uint8_t; };

template <int kBytes>
__device__ __forceinline__ void copy_part(const char* __restrict__ from, char* __restrict__ to, int bytes, int tid) {
  using W = typename Word<kBytes>::type;
  const W* a = reinterpret_cast<const W*>(from);
  W* b = reinterpret_cast<W*>(to);
  const int n = bytes / kBytes;
#pragma unroll 4
  for (int i = tid; i < n; i += kReorderThreads) b[i] = a[i];
}

__global__ void __launch_bounds__(kReorderThreads)
beam_reorder_kernel(const int64_t* __restrict__ slots, const int64_t* __restrict__ parents, int64_t* __restrict__ new_slots, int groups, int beams,
                    int64_t n_slots, const __grid_constant__ Pools pools) {
  // {from, to}: one a beam at most, in the order of the beams, which is the same in every CTA
  extern __shared__ int2 s_copy[];
  uint8_t* const s_parent = reinterpret_cast<uint8_t*>(s_copy + groups * beams);
  __shared__ int s_counts[kReorderThreads / 32];
  constexpr uint8_t kNobody = 255;
  const int tid = threadIdx.x, all = groups * beams;
  for (int i = tid; i < all; i += kReorderThreads) {
    const int64_t p = parents[i];
    s_parent[i] = p >= 0 && p < beams ? uint8_t(p) : kNobody;
  }
  __syncthreads();
  // A thread goes through a group: beams with children, and children that keep a slot, are sets of at most 64.
  int copies = 0;
  for (int base = 0; base < groups; base += kReorderThreads) {
    const int g = base + tid;
    const int64_t* const own = slots + int64_t(g) * beams;
    const uint8_t* const parent = s_parent + g * beams;
    uint64_t going_on = 0, keeps = 0;
    if (g < groups) {
      for (int k = 0; k < beams; ++k) {
        const int p = parent[k];
        if (p == kNobody || (going_on >> p & 1)) continue;
        going_on |= uint64_t(1) << p;
        keeps |= uint64_t(1) << k;
      }
    }
    // Children that keep none and beams without children are equally many.  f(to, beam, from): from is -1 where nothing is copied.
    auto each = [&](auto f) {
      uint64_t spare = ~going_on;
      for (int k = 0; k < beams; ++k) {
        const int p = parent[k];
        if (keeps >> k & 1) {
          f(own[p], k, int64_t(-1));
          continue;
        }
        const int to = __ffsll(int64_t(spare)) - 1;
        spare &= spare - 1;
        const int64_t t = own[to], from = p == kNobody ? -1 : own[p];
        f(t, k, from < n_slots && t >= 0 && t < n_slots ? from : int64_t(-1));
      }
    };
    int mine = 0;
    if (g < groups) each([&](int64_t to, int k, int64_t from) {
      mine += from >= 0;
      if (blockIdx.x == 0) new_slots[int64_t(g) * beams + k] = to;
    });
    int upto = mine;                                       // sum over the threads up to this one
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const int more = __shfl_up_sync(0xffffffffu, upto, s);
      if (tid % 32 >= s) upto += more;
    }
    __syncthreads();
    if (tid % 32 == 31) s_counts[tid / 32] = upto;
    __syncthreads();
    int at = copies + upto - mine;
#pragma unroll
    for (int w = 0; w < kReorderThreads / 32; ++w) {
      at += w < tid / 32 ? s_counts[w] : 0;
      copies += s_counts[w];
    }
    if (mine) each([&](int64_t to, int, int64_t from) {
      if (from >= 0) s_copy[at++] = make_int2(int(from), int(to));
    });
  }
  __syncthreads();
  const int parts = pools.first_part[pools.n];
  const int64_t work = int64_t(copies) * parts;
  for (int64_t i = blockIdx.x; i < work; i += gridDim.x) {
    const int2 c = s_copy[i / parts];
    const int part = int(i % parts);
    int lo = 0, hi = pools.n;                              // the pool this part is of
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (pools.first_part[mid] <= part) lo = mid; else hi = mid;
    }
    const int64_t bytes = pools.bytes[lo], at = int64_t(part - pools.first_part[lo]) * kReorderPart;
    const int n = int(min64(kReorderPart, bytes - at));
    const char* from = pools.at[lo] + c.x * bytes + at;
    char* to = pools.at[lo] + c.y * bytes + at;
    const uintptr_t off = reinterpret_cast<uintptr_t>(pools.at[lo]) | uintptr_t(bytes);
    if (off % 16 == 0) copy_part<16>(from, to, n, tid);
    else if (off % 4 == 0) copy_part<4>(from, to, n, tid);
    else copy_part<1>(from, to, n, tid);
  }
}

}  // namespace
}  // namespace mb200

using namespace mb200;

extern "C" int64_t mb200_beam_select_scratch_bytes(int64_t groups, int64_t beams, int64_t V, int num) {
  if (groups < 0 || beams < 0 || V < 0 || num < 0) return 0;
  return groups * beams * ((V + kSelSlice - 1) / kSelSlice) * int64_t(sizeof(Slice) + num * sizeof(uint64_t));
}

extern "C" int mb200_beam_select(const void* logits, const float* scores, const uint8_t* finished, void* scratch, float* out_scores,
                                 int64_t* out_tokens, int64_t* out_parents, int64_t groups, int64_t beams, int64_t V, int num, int64_t end_token,
                                 int64_t row_stride, int dtype, void* stream) {
  if (groups < 0 || beams < 1 || V < 1 || num < 1 || num > beams * V) return MB200_EINVAL;
  if (dtype != MB200_F32 && dtype != MB200_BF16) return MB200_EDTYPE;
  if (finished && (end_token < 0 || end_token >= V)) return MB200_EINVAL;
  if (beams > kMostBeams || num > kMostNum || V >= (int64_t(1) << 30) || groups * beams > 65535) return MB200_ETOOBIG;
  if (groups == 0) return MB200_OK;
  if (!logits || !scores || !scratch || !out_scores || !out_tokens || !out_parents) return MB200_EINVAL;
  if (!aligned16(scratch)) return MB200_EALIGN;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t rows = groups * beams, n_slices = (V + kSelSlice - 1) / kSelSlice;
  if (beams * n_slices * num >= (int64_t(1) << 31)) return MB200_ETOOBIG;
  Slice* slices = static_cast<Slice*>(scratch);
  uint64_t* best = reinterpret_cast<uint64_t*>(slices + rows * n_slices);
  const dim3 grid(static_cast<unsigned>(n_slices), static_cast<unsigned>(rows));
  const bool vec = aligned16(logits) && row_stride * (dtype == MB200_F32 ? 4 : 2) % 16 == 0;
#define MB200_SLICES(TT, VEC) beam_slices_kernel<TT, VEC><<<grid, kSelThreads, 0, st>>>((const TT*)logits, row_stride, int(V), num, slices, best)
  if (dtype == MB200_F32) { if (vec) MB200_SLICES(float, true); else MB200_SLICES(float, false); }
  else { if (vec) MB200_SLICES(__nv_bfloat16, true); else MB200_SLICES(__nv_bfloat16, false); }
#undef MB200_SLICES
  if (const int rc = check_launch()) return rc;
  // started while the slices are still at work, so that its launch costs no time of its own
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t how{};
  how.gridDim = dim3(unsigned(groups)); how.blockDim = dim3(kSelThreads); how.stream = st; how.attrs = &early; how.numAttrs = 1;
  const Slice* slices_c = slices;
  const uint64_t* best_c = best;
  if (cudaLaunchKernelEx(&how, beam_join_kernel, slices_c, best_c, scores, finished, logits, row_stride, dtype, int(beams), int(n_slices), int(V), num,
                         int(end_token), out_scores, out_tokens, out_parents) != cudaSuccess)
    return MB200_ELAUNCH;
  return check_launch();
}

extern "C" int mb200_beam_reorder(const int64_t* slots, const int64_t* parents, int64_t* new_slots, int64_t groups, int64_t beams, int64_t n_slots,
                                  void* const* pools, const int64_t* entry_bytes, int n_pools, void* stream) {
  if (groups < 0 || beams < 0 || n_slots < 0 || n_pools < 0 || (n_pools > 0 && (!pools || !entry_bytes))) return MB200_EINVAL;
  if (groups == 0 || beams == 0) return MB200_OK;
  if (!slots || !parents || !new_slots || new_slots == slots || new_slots == parents) return MB200_EINVAL;
  if (beams > kMostBeams || groups > kMostSlotBeams || groups * beams > kMostSlotBeams || n_slots >= (int64_t(1) << 31)) return MB200_ETOOBIG;
  for (int i = 0; i < n_pools; ++i) {
    if (!pools[i] || entry_bytes[i] < 0) return MB200_EINVAL;
    if (entry_bytes[i] >= (int64_t(1) << 31)) return MB200_ETOOBIG;
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int all = int(groups * beams), shared = all * int(sizeof(int2) + 1);
  int done = 0;
  do {                                                     // one launch takes kMostPools pools
    Pools p{};
    int64_t parts = 0;
    while (done < n_pools && p.n < kMostPools) {
      p.at[p.n] = static_cast<char*>(pools[done]);
      p.bytes[p.n] = entry_bytes[done];
      p.first_part[p.n] = int(parts);
      const int64_t more = (entry_bytes[done] + kReorderPart - 1) / kReorderPart;
      if (parts + more >= (int64_t(1) << 30)) return MB200_ETOOBIG;
      parts += more;
      ++p.n; ++done;
    }
    p.first_part[p.n] = int(parts);
    // at most one copy a beam but a group's first
    const int64_t most = (groups * (beams - 1)) * parts;
    const unsigned ctas = unsigned(most < 1 ? 1 : min64(most, int64_t(sm_count()) * 8));
    beam_reorder_kernel<<<ctas, kReorderThreads, shared, st>>>(slots, parents, new_slots, int(groups), int(beams), n_slots, p);
    if (const int rc = check_launch()) return rc;
  } while (done < n_pools);
  return MB200_OK;
}
