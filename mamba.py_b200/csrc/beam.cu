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
// different beams come that close, which is a few groups in a hundred calls, the joining CTA sums those beams' exponentials again in 64 bits.

constexpr int kSelPer = 16;                                // logits of a thread at a time
constexpr int kMostNum = 64, kMostBeams = 64;
constexpr int kCheck = 4;                                  // chunks after which the list is looked at

// By how much two logsumexps may be apart for rounding alone.  An exponent t = (v - top) log2(e) is off by 2.25 x 2^-24 |t| (a difference, a product,
// a constant), and the mean of |t| under the softmax is at most log2 of the vocabulary; it goes to the thread's maximum, from there to the CTA's and
// to the beam's, 3 steps that share |t|, with an ex2.approx of 2^-22 each (a new maximum of the thread is one more, at worst once a chunk, of which all
// but the last then count for little); a thread adds 16 logits in fours; all further sums are in 64 bits.  In units of 2^-24, twice:
__device__ __forceinline__ double too_close(int V) {
  return 2 * 0x1p-24 * (2.25 * 0.6931472 * log2(double(V)) + 4. * 4 + 5.);
}

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

// The lanes' values in falling order.
__device__ __forceinline__ uint32_t sorted_in_warp(uint32_t x, int lane) {
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int step = size / 2; step >= 1; step >>= 1) {
      const uint32_t other = __shfl_xor_sync(0xffffffffu, x, step);
      x = ((lane & step) == 0) == ((lane & size) == 0) ? max(x, other) : min(x, other);
    }
  return x;
}

// How the highest are found.  A warp in which num lanes hold a value as high as K holds num that high, and so do the CTA's warps together if
// each has its share of lanes that high; so no logit below K is wanted.  The higher of the two, over the slice's first chunk and the threads' own
// highest, is K.  Whatever reaches K, in the chunks that follow too (about num a chunk, if they are alike), is put side by side with its place, and
// every item counts those ahead of it; between chunks the num-th of them becomes the new K.  That may be a
// value that very many logits share (a mask's): equal to K, then, counts only up to the num-th place that does, of which there are num in the
// first chunk or none.  Should a chunk have more than there is room for all the same (ascending logits may, and a first chunk that a mask empties makes
// the next one), num rounds over the slice find the highest.
// Bound: 6 instructions a logit that it cannot do without (load and conversion, maximum, half of a difference, product and sum, ex2) would take about as
// long as its 2 bytes from HBM.  It executes 18 (288 a warp for 512 logits: bounds, thresholds, sort and counts are the others) at half the issue slots and
// takes 4 times as long as the bytes, some 2 us of a CTA's time for the first chunk's sort and the counts at the end.  So a CTA takes as many chunks as leave
// 1024 threads for every SM, with the next chunk's loads in flight.  64 x 4 x 50280 in bfloat16: 58 us with a CTA to every 8192 logits and a count of
// all threads' highest, 25 with the warps' sort, 22 with several chunks a CTA, 18 with the join's work and the exponentials' in pairs.
template <typename T, bool kVec, int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads)
beam_slices_kernel(const T* __restrict__ logits, int64_t stride, int V, int slice, int num, Slice* __restrict__ slices, uint64_t* __restrict__ best) {
  constexpr int kWarps = kThreads / 32, kChunk = kThreads * kSelPer, kList = 4 * kThreads;      // kList: items side by side in shared memory
  __shared__ uint64_t s_list[kList], s_best[kMostNum], s_key[kWarps];
  __shared__ uint32_t s_least[2][kWarps];
  __shared__ float s_top[kWarps];
  __shared__ double s_sum[kWarps];
  __shared__ int s_n;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t row = blockIdx.y, part = row * gridDim.x + blockIdx.x;
  const int v0 = int(blockIdx.x) * slice, v1 = min(V, v0 + slice);
  const T* p = logits + row * stride;
  if (tid == 0) s_n = 0;
  cudaTriggerProgrammaticLaunchCompletion();               // the joining kernel may start, and waits for this one's end
  constexpr int kE = kVec ? Elem<T>::kVec : 1, kLoads = kSelPer / kE;
  struct alignas(sizeof(T) * kE) Raw { T v[kE]; };
  auto at = [&](int c0, int j) { return c0 + ((j / kE) * kThreads + tid) * kE + j % kE; };
  auto fetch = [&](int c0, Raw (&raw)[kLoads]) {
    if (kVec && c0 + kChunk <= v1) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i)
        if constexpr (kVec) *reinterpret_cast<uint4*>(&raw[i]) = __ldcs(reinterpret_cast<const uint4*>(p + at(c0, i * kE)));
      return;
    }
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int c = at(c0, i * kE);
      if (kVec && c + kE <= v1) {
        if constexpr (kVec) *reinterpret_cast<uint4*>(&raw[i]) = __ldcs(reinterpret_cast<const uint4*>(p + c));
      } else {
#pragma unroll
        for (int k = 0; k < kE; ++k) raw[i].v[k] = c + k < v1 ? p[c + k] : Elem<T>::from_f(-INFINITY);
      }
    }
  };
  // num highest of the list, highest first, in s_best
  auto rank = [&](int n) {
    for (int i = tid; i < n; i += kThreads) {
      const uint64_t key = s_list[i];
      int ahead = 0;
#pragma unroll 4
      for (int k = 0; k < n; ++k) ahead += s_list[k] > key;
      if (ahead < num) s_best[ahead] = key;
    }
    __syncthreads();
  };
  Raw raw[kLoads];
  fetch(v0, raw);
  float least = -INFINITY;                                 // K
  int within = v1;                                         // equal to K counts below this place
  float mine = -INFINITY;                                  // the thread's maximum,
  double all = 0.;                                         // and its sum of exp(logit - maximum)
  bool room = true;
  for (int c0 = v0, chunk = 0; c0 < v1; c0 += kChunk, ++chunk) {
    float v[kSelPer];
#pragma unroll
    for (int j = 0; j < kSelPer; j += 2) {
      if constexpr (kVec) {
        const float2 two = pair_f(&raw[j / kE].v[j % kE]);
        v[j] = two.x; v[j + 1] = two.y;
      } else {
        v[j] = Elem<T>::to_f(raw[j].v[0]); v[j + 1] = Elem<T>::to_f(raw[j + 1].v[0]);
      }
    }
    if (c0 + kChunk < v1) fetch(c0 + kChunk, raw);
    float high = -INFINITY, high2 = -INFINITY;             // of the halves
#pragma unroll
    for (int j = 0; j < kSelPer / 2; ++j) {
      high = fmaxf(high, v[j]);
      high2 = fmaxf(high2, v[kSelPer / 2 + j]);
    }
    if (chunk == 0) {
      // (with more than 32 wanted, the halves' lowest stands for 64 lanes)
      const uint32_t x = sorted_in_warp(order_of(fmaxf(high, high2)), lane);
      uint32_t whole = __shfl_sync(0xffffffffu, x, (num <= 32 ? num : 32) - 1);
      if (num > 32) whole = __reduce_min_sync(0xffffffffu, order_of(fminf(high, high2)));
      const uint32_t share = __shfl_sync(0xffffffffu, x, (num + kWarps - 1) / kWarps - 1);
      if (lane == 0) {
        s_least[0][warp] = whole;
        s_least[1][warp] = share;
      }
      __syncthreads();
      uint32_t most = 0, all = ~0u;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        most = max(most, s_least[0][w]);
        all = min(all, s_least[1][w]);
      }
      least = value_of(max(most, all));
      // The usual number of logits this high is little more than num.  If many are equal to K, the num-th place that is closes it for the others.
      int equal = 0;
#pragma unroll
      for (int j = 0; j < kSelPer; ++j) equal += v[j] == least && at(c0, j) < v1;
      if (__syncthreads_or(equal > 2)) {
        // places are in the order of load, thread and element: counted load by load
        int before = 0;
        for (int i = 0; i < kLoads; ++i) {
          int n = 0;
#pragma unroll
          for (int j = 0; j < kSelPer; ++j) n += j / kE == i && v[j] == least && at(c0, j) < v1;
          int upto = n;
#pragma unroll
          for (int s = 1; s < 32; s <<= 1) {
            const int more = __shfl_up_sync(0xffffffffu, upto, s);
            if (lane >= s) upto += more;
          }
          __syncthreads();
          if (lane == 31) s_least[0][warp] = upto;
          __syncthreads();
          int total = 0;
          for (int w = 0; w < kWarps; ++w) {
            if (w < warp) upto += s_least[0][w];
            total += s_least[0][w];
          }
          int rank_of = before + upto - n;
#pragma unroll
          for (int j = 0; j < kSelPer; ++j)
            if (j / kE == i && v[j] == least && at(c0, j) < v1 && rank_of++ == num - 1) s_n = -at(c0, j) - 1;
          before += total;
        }
        __syncthreads();
        if (s_n < 0) within = -s_n;                        // behind the num-th such place
        __syncthreads();
        if (tid == 0) s_n = 0;
        __syncthreads();
      }
    }
    const float top = fmaxf(mine, fmaxf(high, high2));
    if (top > mine) {
      all *= double(ex2f((mine - top) * kLog2e));          // (0 from -inf)
      mine = top;
    }
    const float from = top == -INFINITY ? 0.f : top;
    float2 sums[2];
#pragma unroll
    for (int j = 0; j < kSelPer; j += 2) {
      const float2 t = __fmul2_rn(__fadd2_rn(make_float2(v[j], v[j + 1]), make_float2(-from, -from)), make_float2(kLog2e, kLog2e));
      const float2 x = make_float2(ex2f(t.x), ex2f(t.y));
      sums[j / 2 % 2] = j < 4 ? x : __fadd2_rn(sums[j / 2 % 2], x);
    }
    all += double((sums[0].x + sums[0].y) + (sums[1].x + sums[1].y));
    // Few threads look at their logits one by one, and read those that count again: a body for each of the 16 would cost more than all the rest.
    if (fmaxf(high, high2) >= least) {
      unsigned hits = 0;
#pragma unroll
      for (int j = 0; j < kSelPer; ++j) hits |= unsigned(v[j] >= least) << j;
#pragma unroll 1
      for (; hits; hits &= hits - 1) {
        const int c = at(c0, __ffs(int(hits)) - 1);
        const float x = c < v1 ? Elem<T>::to_f(p[c]) : -INFINITY;
        if (c >= (x == least ? within : v1)) continue;
        const int n = atomicAdd(&s_n, 1);
        if (n < kList) s_list[n] = key_of(x, c);
      }
    }
    if (c0 + kChunk >= v1) break;
    if (chunk % kCheck != 0) continue;
    __syncthreads();
    const int n = s_n;
    if (n > kList) {
      room = false;
    } else if (n > 2 * num && room) {
      rank(n);
      if (tid < num) s_list[tid] = s_best[tid];
      if (tid == 0) s_n = num;
      // places only rise from here on, so nothing equal to the num-th of these is wanted any more
      least = value_of(uint32_t(s_best[num - 1] >> 32));
      within = 0;
    }
    __syncthreads();
  }
  float top = mine;
#pragma unroll
  for (int s = 16; s >= 1; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
  if (lane == 0) s_top[warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_top[w]);
  if (top > -INFINITY) all *= double(ex2f((mine - top) * kLog2e));
#pragma unroll
  for (int s = 16; s >= 1; s >>= 1) all += __shfl_xor_sync(0xffffffffu, all, s);
  if (lane == 0) s_sum[warp] = all;
  const int n = s_n;
  uint64_t* const out = best + part * num;
  if (room && n <= kList) {
    rank(n);
    for (int i = tid; i < num; i += kThreads) out[i] = i < n ? s_best[i] : 0;
  } else {
    uint64_t last = ~uint64_t(0);
    for (int r = 0; r < num; ++r) {
      uint64_t key = 0;
      for (int c = v0 + tid; c < v1; c += kThreads) {
        const uint64_t k = key_of(Elem<T>::to_f(p[c]), c);
        if (k < last) key = max64(key, k);
      }
#pragma unroll
      for (int s = 16; s >= 1; s >>= 1) key = max64(key, __shfl_xor_sync(0xffffffffu, key, s));
      __syncthreads();
      if (lane == 0) s_key[warp] = key;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kWarps; ++w) key = max64(key, s_key[w]);
      if (tid == 0) out[r] = key;
      last = key;
    }
  }
  if (tid == 0) {
    all = 0.;
    for (int w = 0; w < kWarps; ++w) all += s_sum[w];
    slices[part] = Slice{top, 0.f, all};
  }
}

// One CTA a group.  Every slice lists its highest in falling order, so candidates are taken by their rank in the lists, all lists' first ones first, as many
// ranks at a time as the threads can take; once a whole rank holds nothing ahead of the num-th highest so far, no further one does.  What
// the argument above on lanes and warps does not rule out goes side by side in shared memory, where each counts those ahead of it.
// Bound by latency: two round trips to global memory, a logarithm in 64 bits, and three or four barriers for every set of ranks (one or two sets in
// general).  16 groups of 16 beams of 128256, 32 of them: 38 us for both kernels, where the join alone took 61 with all 1024 candidates
// of a group in any order.
template <int kThreads>
__global__ void __launch_bounds__(kThreads)
beam_join_kernel(const Slice* __restrict__ slices, const uint64_t* __restrict__ best, const float* __restrict__ scores,
                 const uint8_t* __restrict__ finished, const void* __restrict__ logits, int64_t stride, int dtype, int beams, int n_slices, int V,
                 int num, int end_token, float* __restrict__ out_scores, int64_t* __restrict__ out_tokens, int64_t* __restrict__ out_parents) {
  constexpr int kWarps = kThreads / 32;
  __shared__ double s_total[kMostBeams];                   // logsumexp of a beam's logits less their maximum (which may be far beyond it)
  __shared__ float s_score[kMostBeams], s_top[kMostBeams];
  __shared__ uint8_t s_kind[kMostBeams];
  __shared__ double s_sum[kWarps];
  // an item: the value's order in 64 bits, and beam << 32 | token
  __shared__ uint64_t s_order[kThreads + kMostNum], s_place[kThreads + kMostNum], s_best[2][kMostNum];
  __shared__ uint32_t s_least[2][kWarps], s_close[kMostBeams / 32];       // beams that are too close to one another
  __shared__ int s_n;
  enum { kOpen, kFinished, kDead };
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t g = blockIdx.x;
  // Lists of the group, and how a set of candidates is made of them: whole ranks of all lists, or a part of one.
  const int lists = beams * n_slices, ranks = lists <= kThreads ? kThreads / lists : 1, parts = (lists + kThreads - 1) / kThreads;
  const int sets = parts > 1 ? num * parts : (num + ranks - 1) / ranks;
  // (a list's ranks side by side, so that every warp has some of the first ones)
  const int my_list = tid / ranks, my_rank = tid % ranks;
  auto list_of = [&](int set) { return parts > 1 ? set % parts * kThreads + tid : my_list; };
  auto rank_of = [&](int set) { return parts > 1 ? set / parts : set * ranks + my_rank; };
  const uint64_t* const mine = best + g * lists * num;
  auto fetch = [&](int set) -> uint64_t {
    const int l = list_of(set), r = rank_of(set);
    return l < lists && r < num ? mine[int64_t(l) * num + r] : 0;
  };
  cudaGridDependencySynchronize();
  const uint64_t first_key = fetch(0);
  for (int k = warp; k < beams; k += kWarps) {          // a warp a beam
    const int64_t row = g * beams + k;
    const Slice* const part = slices + row * n_slices;
    Slice one{-INFINITY, 0.f, 0.};
    if (lane < n_slices) one = part[lane];
    const float score = scores[row];
    const bool done = finished && finished[row];
    float top = one.top;
    for (int i = lane + 32; i < n_slices; i += 32) top = fmaxf(top, part[i].top);
#pragma unroll
    for (int s = 16; s >= 1; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
    double sum = one.sum * double(ex2f((one.top - top) * kLog2e));
    for (int i = lane + 32; i < n_slices; i += 32) sum += part[i].sum * double(ex2f((part[i].top - top) * kLog2e));
#pragma unroll
    for (int s = 16; s >= 1; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
    if (lane == 0) {
      s_total[k] = log(sum);
      s_score[k] = score;
      s_top[k] = top;
      s_kind[k] = uint8_t(!isfinite(score) ? kDead : done ? kFinished : isfinite(top) && isfinite(sum) ? kOpen : kDead);
    }
  }
  if (tid == 0) s_n = 0;
  if (tid < kMostBeams / 32) s_close[tid] = 0;
  __syncthreads();
  // The thread's candidate of a set: order (0: none) and place.  What is no candidate stands in at -inf, lowest tokens first: of those, a slice lists
  // enough among its highest logits if it has fewer than num others, and if one has not, no stand-in is needed.
  const uint64_t nothing = order_of(-double(INFINITY));
  auto candidate = [&](int set, uint64_t& place) -> uint64_t {
    const int l = list_of(set), r = rank_of(set);
    if (l >= lists || r >= num) return 0;
    const int k = l / n_slices, kind = s_kind[k];
    place = uint64_t(k) << 32;
    if (kind == kOpen) {
      const uint64_t key = set == 0 ? first_key : mine[int64_t(l) * num + r];
      place |= uint32_t(~uint32_t(key));
      return key ? order_of(double(s_score[k]) + ((double(value_of(uint32_t(key >> 32))) - double(s_top[k])) - s_total[k])) : 0;
    }
    if (l != k * n_slices) return 0;                       // the first slice's list stands for such a beam
    int t = r;
    if (kind == kFinished) {
      if (r == 0) {
        place |= uint32_t(end_token);
        return order_of(double(s_score[k]));
      }
      if (--t >= end_token) ++t;
    }
    place |= uint32_t(t);
    return t < V ? nothing : 0;
  };
  for (bool again = false;; again = true) {
    uint64_t least_order = 0, least_place = 0;             // of the num-th highest so far
    bool fresh = false;                                    // something of this rank went into the list
    uint64_t first_order = 0, first_place = 0;             // the thread's candidate of the first set
    for (int set = 0; set < sets; ++set) {
      uint64_t place = 0;
      const uint64_t order = candidate(set, place);
      if (set == 0) first_order = order, first_place = place;
      const uint32_t high = uint32_t(order >> 32);
      const uint32_t sorted = sorted_in_warp(high, lane);
      if (lane == (num <= 32 ? num : 32) - 1) s_least[0][warp] = num <= 32 ? sorted : 0;
      if (lane == (num + kWarps - 1) / kWarps - 1) s_least[1][warp] = sorted;
      __syncthreads();
      uint32_t most = 0, all = ~0u;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        most = max(most, s_least[0][w]);
        all = min(all, s_least[1][w]);
      }
      const bool in = order && high >= max(most, all) && (order > least_order || (order == least_order && place < least_place));
      const unsigned who = __ballot_sync(0xffffffffu, in);
      int base = 0;
      if (lane == 0 && who) base = atomicAdd(&s_n, __popc(who));
      base = __shfl_sync(0xffffffffu, base, 0);
      if (in) {
        const int n = base + __popc(who & ((1u << lane) - 1));
        s_order[n] = order;
        s_place[n] = place;
      }
      __syncthreads();
      const int n = s_n, kept = least_order ? num : 0;
      fresh = (parts > 1 && set % parts != 0 && fresh) || n > kept || !least_order;
      if (n > kept) {
        // the lanes of a group of 8 count their eighths of what is ahead of a candidate (one thread a candidate: 62 candidates take 4 us)
        for (int first = 0; first < n; first += kThreads / 8) {
          const int i = first + tid / 8;
          const uint64_t o = i < n ? s_order[i] : 0, q = i < n ? s_place[i] : 0;
          int ahead = 0;
#pragma unroll 4
          for (int k = tid % 8; k < n; k += 8) {
            const uint64_t other = s_order[k], where = s_place[k];
            ahead += int(other > o) | (int(other == o) & int(where < q));
          }
#pragma unroll
          for (int s = 4; s >= 1; s >>= 1) ahead += __shfl_xor_sync(0xffffffffu, ahead, s);
          if (i < n && tid % 8 == 0 && ahead < num) {
            s_best[0][ahead] = o;
            s_best[1][ahead] = q;
          }
        }
        __syncthreads();
        const int left = min(n, num);
        if (tid < left) {
          s_order[tid] = s_best[0][tid];
          s_place[tid] = s_best[1][tid];
        }
        if (tid == 0) s_n = left;
        if (left == num) {
          least_order = s_best[0][num - 1];
          least_place = s_best[1][num - 1];
        }
      }
      __syncthreads();
      if (!fresh && (parts == 1 || set % parts == parts - 1)) break;
    }
    if (again) break;
    // Whether 32 bits cannot tell candidates of different beams apart.  Neighbours among the chosen, and the last of them with those behind it,
    // say it of all: between two that are too close, each is too close to the next.
    bool close = false;
    const double apart = too_close(V), last = value_of(s_best[0][num - 1]);
    const int last_beam = int(s_best[1][num - 1] >> 32);
    auto compare = [&](int k, int other) {
      if (k == other || (s_kind[k] != kOpen && s_kind[other] != kOpen)) return;
      close = true;
      atomicOr(&s_close[k / 32], 1u << k % 32);
      atomicOr(&s_close[other / 32], 1u << other % 32);
    };
    if (tid < num - 1) {
      const double value = value_of(s_best[0][tid + 1]);
      if (value > -INFINITY && value_of(s_best[0][tid]) - value <= apart) compare(int(s_best[1][tid] >> 32), int(s_best[1][tid + 1] >> 32));
    }
    for (int set = 0; set < sets; ++set) {
      uint64_t place = first_place;
      const uint64_t order = set == 0 ? first_order : candidate(set, place);
      const double value = value_of(order);
      const bool near = order && value > -INFINITY && last - value <= apart;
      if (near && (order < least_order || (order == least_order && place > least_place))) compare(int(place >> 32), last_beam);
      if (parts == 1 && (set + 1 == sets || !__syncthreads_or(near))) break;
    }
    if (!__syncthreads_or(close)) break;
    for (int k = 0; k < beams; ++k) {
      if (s_kind[k] != kOpen || !(s_close[k / 32] >> k % 32 & 1u)) continue;
      const int64_t from = (g * beams + k) * stride;
      const double top = s_top[k];
      double sum = 0.;
      for (int v = tid; v < V; v += kThreads) {
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
        for (int w = 0; w < kWarps; ++w) sum += s_sum[w];
        s_total[k] = log(sum);
      }
    }
    if (tid == 0) s_n = 0;
    __syncthreads();
  }
  if (tid < num) {
    out_scores[g * num + tid] = float(value_of(s_best[0][tid]));
    out_parents[g * num + tid] = int64_t(s_best[1][tid] >> 32);
    out_tokens[g * num + tid] = int64_t(uint32_t(s_best[1][tid]));
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
constexpr int kReorderThreads = 256, kReorderPart = 8192;
// (bytes a CTA copies at a time: 64 layers, 24 states of 328 KB, us with 4 / 8 / 16 / 32 / 64 KB 250 / 190 / 194 / 196 / 197)
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

// Logits of a CTA: whole chunks, as many as leave about four CTAs (of 256 threads, two of 512) for every SM.
struct SelectPlan {
  int threads, join_threads;
  int64_t slice, n_slices;
  SelectPlan(int64_t rows, int64_t beams, int64_t V, int num) {
    auto chunks = [&](int t) { return (V + t * kSelPer - 1) / (t * kSelPer); };
    // Where CTAs of 256 threads take several chunks, 512 find a better threshold in their first one (us with 256 / 512: 64 x 4 x 50280, 4 of
    // them 17.9 / 18.0; 16 x 16 x 128256, 32 of them 55 / 43); where not, they halve the CTAs (5 x 32001 9.0 / 10.4).
    threads = rows * chunks(256) > int64_t(sm_count()) * 4 ? 512 : 256;
    const int64_t all = chunks(threads), wanted = int64_t(sm_count()) * (1024 / threads) / (rows > 0 ? rows : 1), slices = wanted < 1 ? 1 : min64(wanted, all);
    slice = (all + slices - 1) / slices * threads * kSelPer;
    n_slices = (V + slice - 1) / slice;
    // A thread a candidate at a time: 8 x 4 of them 18.0 us with 256, 19.1 with 512; 40 x 10 9.8 and 9.0, 32 x 32 43 and 38.
    join_threads = beams * n_slices * num > 256 ? 512 : 256;
  }
};

extern "C" int64_t mb200_beam_select_scratch_bytes(int64_t groups, int64_t beams, int64_t V, int num) {
  if (groups < 1 || beams < 1 || V < 1 || num < 1) return 0;
  return groups * beams * SelectPlan(groups * beams, beams, V, num).n_slices * int64_t(sizeof(Slice) + num * sizeof(uint64_t));
}

extern "C" int mb200_beam_select(const void* logits, const float* scores, const uint8_t* finished, void* scratch, float* out_scores,
                                 int64_t* out_tokens, int64_t* out_parents, int64_t groups, int64_t beams, int64_t V, int num, int64_t end_token,
                                 int64_t row_stride, int dtype, void* stream) {
  if (groups < 0 || beams < 1 || V < 1 || num < 1) return MB200_EINVAL;
  if (dtype != MB200_F32 && dtype != MB200_BF16) return MB200_EDTYPE;
  if (finished && (end_token < 0 || end_token >= V)) return MB200_EINVAL;
  if (beams > kMostBeams || num > kMostNum || V >= (int64_t(1) << 30) || groups > 65535 || groups * beams > 65535) return MB200_ETOOBIG;
  if (num > beams * V) return MB200_EINVAL;
  if (groups == 0) return MB200_OK;
  if (!logits || !scores || !scratch || !out_scores || !out_tokens || !out_parents) return MB200_EINVAL;
  if (!aligned16(scratch)) return MB200_EALIGN;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t rows = groups * beams;
  const SelectPlan plan(rows, beams, V, num);
  const int64_t slice = plan.slice, n_slices = plan.n_slices;
  if (beams * n_slices * num >= (int64_t(1) << 31)) return MB200_ETOOBIG;
  Slice* slices = static_cast<Slice*>(scratch);
  uint64_t* best = reinterpret_cast<uint64_t*>(slices + rows * n_slices);
  const dim3 grid(static_cast<unsigned>(n_slices), static_cast<unsigned>(rows));
  const bool vec = aligned16(logits) && row_stride * (dtype == MB200_F32 ? 4 : 2) % 16 == 0;
#define MB200_SLICES(TT, VEC)                                                                                                                   \
  (plan.threads == 512 ? beam_slices_kernel<TT, VEC, 512> : beam_slices_kernel<TT, VEC, 256>)<<<grid, unsigned(plan.threads), 0, st>>>(         \
      (const TT*)logits, row_stride, int(V), int(slice), num, slices, best)
  if (dtype == MB200_F32) { if (vec) MB200_SLICES(float, true); else MB200_SLICES(float, false); }
  else { if (vec) MB200_SLICES(__nv_bfloat16, true); else MB200_SLICES(__nv_bfloat16, false); }
#undef MB200_SLICES
  if (const int rc = check_launch()) return rc;
  // started while the slices are still at work, so that its launch costs no time of its own
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t how{};
  how.gridDim = dim3(unsigned(groups)); how.blockDim = dim3(unsigned(plan.join_threads)); how.stream = st; how.attrs = &early; how.numAttrs = 1;
  const Slice* slices_c = slices;
  const uint64_t* best_c = best;
  if (cudaLaunchKernelEx(&how, plan.join_threads == 512 ? beam_join_kernel<512> : beam_join_kernel<256>, slices_c, best_c, scores, finished, logits, row_stride, dtype, int(beams), int(n_slices), int(V), num,
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
