// Depthwise causal conv1d + SiLU (d_conv = 4) over sequences of different lengths laid end to end, forward and backward:
//     y[t,e] = silu( bias[e] + sum_k w[e,k] * in(t-3+k, e) ),   in = x within the sequence of row t,
// and before its first row 0 or, when the sequence resumes, the window that its slot holds.  Streaming: what it has to do is to read x and write y
// once.
//
// Where sequences begin is a bit per row.  Rows in front of which none begins, which is nearly all of them, take a path without tests.
#include <type_traits>
#include "conv1d.cuh"
#include "packed.cuh"
#include "tma.cuh"

namespace mb200 {
namespace {

constexpr int kPkThreads = 256, kPkWarps = kPkThreads / 32, kPkResident = 3;
constexpr int kPkChunk = 32, kPkGroup = 8;              // rows of a warp; rows whose loads go out together

// Where sequences begin: a bit for every row from `base` on.
struct Firsts {
  const unsigned* bits;
  int base;
  // of 32 rows from t on, lowest first
  __device__ __forceinline__ unsigned from(int t) const {
    const int at = t - base;
    return __funnelshift_r(bits[at >> 5], bits[(at >> 5) + 1], at & 31);
  }
};

// Of a pool of windows (n_slots, ED, 3): the windows of V neighbouring channels from e on, oldest input first.
template <typename T, int V, int W>
__device__ __forceinline__ void load_window(const T* p, Pk<W> (&win)[V / W][kConvK - 1]) {
  float v[V * 3];
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    const CVec<T, V> q = cload<T, V>(p + k * V, true);
#pragma unroll
    for (int i = 0; i < V; ++i) v[k * V + i] = Elem<T>::to_f(q.v[i]);
  }
#pragma unroll
  for (int i = 0; i < V / W; ++i)
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      if constexpr (W == 1) win[i][k].v = v[3 * i + k];
      else win[i][k].v = make_float2(v[6 * i + k], v[6 * i + 3 + k]);
    }
}

// The last three inputs of sequence r, whose first row is t, for V neighbouring channels; `old`: what is there counts.
template <typename T, int V>
__device__ __forceinline__ void leave_window(const Packed& seqs, int r, int t, bool old, const T* x, int64_t x_sl, T* at) {
  const int n = seqs.end(r, t) - t;
  T u[kConvK - 1][V];
#pragma unroll
  for (int k = 0; k < kConvK - 1; ++k) {
    const int place = n - (kConvK - 1) + k;               // of the input that goes to entry k
#pragma unroll
    for (int i = 0; i < V; ++i) u[k][i] = Elem<T>::from_f(0.f);
    if (place >= 0) {
      const CVec<T, V> in = cload<T, V>(x + int64_t(t + place) * x_sl, true);
#pragma unroll
      for (int i = 0; i < V; ++i) u[k][i] = in.v[i];
    } else if (old) {                                     // shorter than the window: what was there moves up
#pragma unroll
      for (int i = 0; i < V; ++i) u[k][i] = at[3 * i + n + k];
    }
  }
  CVec<T, V> out[kConvK - 1];
#pragma unroll
  for (int j = 0; j < (kConvK - 1) * V; ++j) out[j / V].v[j % V] = u[j % 3][j / 3];
#pragma unroll
  for (int k = 0; k < kConvK - 1; ++k) cstore<T, V>(at + k * V, out[k]);
}

// The thread that meets a sequence's first row also leaves the window, when it is done with its rows: the only one that reads what the slot held.  So
// the (at most two) rows after a first row that need it too, when they fall into the next chunk, are done by the chunk of the first row.
// This form takes any strides, with one channel a thread; the tensor-map form below takes the others.  A warp finds out by itself which sequences
// begin in its rows, a lane a sequence, while the first rows and the filter are on their way: no barrier, and for up to 32 sequences one load.
template <typename T>
__global__ void __launch_bounds__(kPkThreads, kPkResident)
conv1d_silu_packed_fwd_kernel(const Packed seqs, const T* __restrict__ x, const float* __restrict__ w, const float* __restrict__ bias,
                              T* __restrict__ y, T* windows, int64_t ED, int64_t x_sl, int64_t y_sl, int chunks) {
  constexpr int V = 1, kG = kPkGroup;
  constexpr int kBefore = kConvK - 2, kSeen = kBefore + kPkChunk + kConvK - 2;
  struct Begins { int64_t slot; int seq; bool old; };     // a sequence, its slot or -1, and whether it resumes
  __shared__ Begins s_begins[kPkWarps][kSeen];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int begin = (int(blockIdx.x) * kPkWarps + warp) * kPkChunk * chunks, end = int(min64(int64_t(begin) + kPkChunk * chunks, seqs.rows));
  const int64_t e = (int64_t(blockIdx.y) * 32 + lane) * V;
  const bool works = e < ED;
  constexpr int W = (V % 2 == 0) ? 2 : 1, P = V / W;
  using F = Pk<W>;
  F wk[P][kConvK], bv[P], win[P][kConvK - 1];
  CVec<T, V> front[kConvK - 1], v[kG];
  Begins* const mine = s_begins[warp];
  const int tail = seqs.start(seqs.sequences);            // rows from here on belong to no sequence
  if (works) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      bv[i] = bias ? F::load(bias + e + W * i, 1) : F::splat(0.f);
#pragma unroll
      for (int k = 0; k < kConvK; ++k) wk[i][k] = F::load(w + (e + W * i) * kConvK + k, kConvK);
    }
  }
#pragma unroll 1
  for (int t0 = begin; t0 < end; t0 += kPkChunk) {
    const int t1 = min(t0 + kPkChunk, seqs.rows);
    const T* xp = x + int64_t(t0) * x_sl + e;
    if (works) {
#pragma unroll
      for (int k = 0; k < kConvK - 1; ++k) front[k] = cload<T, V>(xp + (k - (kConvK - 1)) * x_sl, t0 + k >= kConvK - 1);
#pragma unroll
      for (int j = 0; j < kG; ++j) v[j] = cload<T, V>(xp + j * x_sl, t0 + j < t1);
    }
    // bit i: a sequence begins at row t0 - 2 + i
    __syncwarp();                                           // (the last chunk's are read)
    uint64_t firsts = 0;
    for (int r = lane; r < seqs.sequences; r += 32) {
      const int first = seqs.start(r), at = first - t0 + kBefore;
      if (at >= 0 && at < kSeen && seqs.end(r, first) > first) {
        firsts |= uint64_t(1) << at;
        mine[at] = Begins{windows ? seqs.slot(r) : -1, r, seqs.resumes(r)};
      }
    }
    __syncwarp();
    firsts = uint64_t(__reduce_or_sync(0xffffffffu, unsigned(firsts))) | uint64_t(__reduce_or_sync(0xffffffffu, unsigned(firsts >> 32))) << 32;
    if (!works) continue;
    T* yp = y + int64_t(t0) * y_sl + e;
    auto enter = [&]() {
#pragma unroll
      for (int k = 0; k < kConvK - 1; ++k) {
        F xv[P];
        unpack<T, V, W>(front[k], xv);
#pragma unroll
        for (int i = 0; i < P; ++i) win[i][k] = xv[i];
      }
    };
    // y of one row, whose input enters the window
    auto row = [&](const CVec<T, V>& q) {
      F xn[P], o[P];
      unpack<T, V, W>(q, xn);
#pragma unroll
      for (int i = 0; i < P; ++i) {
        F acc = pfma(wk[i][0], win[i][0], bv[i]);
        acc = pfma(wk[i][1], win[i][1], acc);
        acc = pfma(wk[i][2], win[i][2], acc);
        acc = pfma(wk[i][3], xn[i], acc);
        win[i][0] = win[i][1]; win[i][1] = win[i][2]; win[i][2] = xn[i];
        o[i] = pmul(acc, psigmoid(acc));
      }
      return pack<T, V, W>(o);
    };
    // No sequence begins in the chunk or in the two rows in front of it, and all of it is rows of sequences.
    if (t0 + kPkChunk <= tail && (firsts & ((uint64_t(1) << (kBefore + kPkChunk)) - 1)) == 0) {
      enter();
#pragma unroll
      for (int g = 0; g < kPkChunk / kG; ++g) {
        if (g > 0) {
#pragma unroll
          for (int j = 0; j < kG; ++j) v[j] = cload<T, V>(xp + j * x_sl, true);
        }
        xp += kG * x_sl;
#pragma unroll
        for (int j = 0; j < kG; ++j) {
          cstore<T, V>(yp, row(v[j]));
          yp += y_sl;
        }
      }
      continue;
    }
    // Rows this chunk does, lo to hi: a row within two of its sequence's first one, if that lies in another chunk, belongs to that chunk.
    auto first_at = [&](int t) { return (firsts >> (t - t0 + kBefore) & 1) != 0; };
    int lo = t0, hi = min(t1, tail);
    constexpr int kFar = -2 * kConvK;
    const int in_front = first_at(t0 - 1) ? t0 - 1 : first_at(t0 - 2) ? t0 - 2 : kFar;
    const int at_end = t1 != t0 + kPkChunk ? kFar : first_at(t1 - 1) ? t1 - 1 : first_at(t1 - 2) ? t1 - 2 : kFar;
    while (lo < t1 && lo - in_front < kConvK - 1 && !first_at(lo)) ++lo;
    while (hi < tail && hi - at_end < kConvK - 1 && !first_at(hi)) ++hi;
    xp += int64_t(lo - t0) * x_sl;
    yp += int64_t(lo - t0) * y_sl;
    if (lo > t0) {
#pragma unroll
      for (int k = 0; k < kConvK - 1; ++k) front[k] = cload<T, V>(xp + (k - (kConvK - 1)) * x_sl, lo + k >= kConvK - 1);
    }
    enter();
#pragma unroll 1
    for (int t = lo; t < hi; t += kG) {
#pragma unroll
      for (int j = 0; j < kG; ++j) v[j] = cload<T, V>(xp + j * x_sl, t + j < hi);
      xp += kG * x_sl;
      if (t + kG <= hi && (firsts >> (t - t0 + kBefore) & ((1u << kG) - 1)) == 0) {
#pragma unroll
        for (int j = 0; j < kG; ++j) {
          cstore<T, V>(yp, row(v[j]));
          yp += y_sl;
        }
        continue;
      }
      // (one row at a time, the others moving up: unrolled, what a first row does eight times over costs the path above its registers)
#pragma unroll 1
      for (int u = t; u < t + kG && u < hi; ++u) {
        if (first_at(u)) {
          const Begins q = mine[u - t0 + kBefore];
          if (q.slot >= 0 && q.old) {
            load_window<T, V, W>(windows + (q.slot * ED + e) * (kConvK - 1), win);
          } else {
#pragma unroll
            for (int i = 0; i < P; ++i)
#pragma unroll
              for (int k = 0; k < kConvK - 1; ++k) win[i][k] = F::splat(0.f);
          }
        }
        cstore<T, V>(yp, row(v[0]));
        yp += y_sl;
#pragma unroll
        for (int j = 0; j + 1 < kG; ++j) v[j] = v[j + 1];
      }
    }
    CVec<T, V> zero;
#pragma unroll
    for (int i = 0; i < V; ++i) zero.v[i] = Elem<T>::from_f(0.f);
    for (int t = max(t0, tail); t < t1; ++t) cstore<T, V>(y + int64_t(t) * y_sl + e, zero);
    if (!windows) continue;
    // What the sequences that begin in this chunk leave.
    for (uint64_t own = firsts >> kBefore & ((uint64_t(1) << kPkChunk) - 1); own; own &= own - 1) {
      const int t = t0 + __ffsll(int64_t(own)) - 1;
      const Begins q = mine[t - t0 + kBefore];
      if (q.slot < 0) continue;
      leave_window<T, V>(seqs, q.seq, t, q.old, x + e, x_sl, windows + (q.slot * ED + e) * (kConvK - 1));
    }
  }
}

// The same for tensors that a tensor map describes.  With loads into registers a warp's are out only while it has nothing to compute, and neither the
// instructions (36 % of the issue slots) nor HBM (half) are busy.  Here a warp does nothing but keep boxes of 32 rows (and the three in front,
// the two behind) by 256 bytes of channels coming, several ahead, and finds where sequences begin in them; four warps take 8 rows of a box
// each, a lane 8 bytes of channels, and store y.  A CTA walks through every gridDim.y-th box of its channels.
// bfloat16, us so / one channel a thread / four: 8000 x 5120, 12 sequences 32.9 / - / 42.2 (a copy 27.4), 16000 x 1536 20.2 / 30.1 / 26.5, 4000 x 1536
// 8.8 / 10.3 / 12.2, 2999 x 1000 7.4 / 6.9 / 9.4, 1000 x 512 4.2 / 5.0 / 9.1.
// Each sigmoid has a reciprocal of its own.  One for the product of a pair's sums saves nothing (8192 x 5120 30.4 and 30.4, the backward at 16000 x 1536
// 38.1 for 39.4), runs out of range far below zero and leaves a sigmoid near 1 a rounding off, which the derivative multiplies with the preactivation.
constexpr int kTcRows = 32, kTcBox = kConvK - 1 + kTcRows + kConvK - 2, kTcBytes = 256, kTcStages = 4, kTcWarps = 4, kTcResident = 5;
constexpr int kTcThreads = 32 * (kTcWarps + 1);

__device__ int g_conv_status = MB200_DEV_OK;

template <typename T>
__global__ void __launch_bounds__(kTcThreads, kTcResident)
conv1d_silu_packed_tma_kernel(const __grid_constant__ CUtensorMap map, const Packed seqs, const T* __restrict__ x,
                              const float* __restrict__ w, const float* __restrict__ bias, T* __restrict__ y, T* windows,
                              int64_t ED, int64_t x_sl, int64_t y_sl) {
  constexpr int kTcChannels = kTcBytes / int(sizeof(T)), V = kTcChannels / 32, W = 2, P = V / W;
  constexpr int kMine = kTcRows / kTcWarps, kBefore = kConvK - 2, kSeen = kBefore + kTcRows + kConvK - 2;
  constexpr int kBytes = kTcBox * kTcBytes;
  static_assert(kBytes % 128 == 0, "boxes stay aligned");
  struct Begins { int64_t slot; int seq; bool old; };     // a sequence, its slot or -1, and whether it resumes
  extern __shared__ __align__(128) unsigned char smem[];  // [kTcStages] boxes
  __shared__ Begins s_begins[kTcStages][kSeen];
  __shared__ uint64_t s_firsts[kTcStages];                // bit i: a sequence begins at row i - 2 of the box's 32
  __shared__ uint64_t full[kTcStages], empty[kTcStages];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t e0 = int64_t(blockIdx.x) * kTcChannels;
  const int boxes = (seqs.rows + kTcRows - 1) / kTcRows;
  if (tid == 0) {
#pragma unroll
    for (int i = 0; i < kTcStages; ++i) { mbar_init(&full[i], 2); mbar_init(&empty[i], kTcWarps); }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  const int tail = seqs.start(seqs.sequences);            // rows from here on belong to no sequence
  int stage = 0, round = 0;
  auto next = [&]() {
    if (++stage == kTcStages) { stage = 0; round ^= 1; }
  };
  if (warp == kTcWarps) {
    int r0 = 0;                                           // sequences in front of it begin in front of the box
    for (int box = blockIdx.y; box < boxes; box += gridDim.y) {
      const int t0 = box * kTcRows;
      if (!mbar_wait(&empty[stage], round ^ 1)) { atomicExch(&g_conv_status, MB200_DEV_WAIT_TIMEOUT); return; }
      if (lane == 0) {
        mbar_expect_tx(&full[stage], kBytes);
        tma_load_3d(smem + stage * kBytes, &map, int(e0), t0 - (kConvK - 1), 0, &full[stage]);
      }
      for (;;) {
        const int r = r0 + lane;
        const int n = __popc(__ballot_sync(0xffffffffu, r < seqs.sequences && seqs.start(r) < t0 - kBefore));
        r0 += n;
        if (n < 32) break;
      }
      uint64_t firsts = 0;
      for (int base = r0;; base += 32) {
        const int r = base + lane, first = r < seqs.sequences ? seqs.start(r) : seqs.rows, at = first - t0 + kBefore;
        const bool in = r < seqs.sequences && at >= 0 && at < kSeen;
        if (in && seqs.end(r, first) > first) {
          firsts |= uint64_t(1) << at;
          s_begins[stage][at] = Begins{windows ? seqs.slot(r) : -1, r, seqs.resumes(r)};
        }
        if (!__all_sync(0xffffffffu, in)) break;          // (offsets that fall are nobody's promise)
      }
      firsts = uint64_t(__reduce_or_sync(0xffffffffu, unsigned(firsts))) | uint64_t(__reduce_or_sync(0xffffffffu, unsigned(firsts >> 32))) << 32;
      if (lane == 0) {
        s_firsts[stage] = firsts;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&full[stage]);
      next();
    }
    return;
  }
  const int64_t e = e0 + lane * V;
  const bool works = e < ED;
  using F = Pk<W>;
  F wk[P][kConvK], bv[P], win[P][kConvK - 1];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    bv[i] = works && bias ? F::load(bias + e + W * i, 1) : F::splat(0.f);
#pragma unroll
    for (int k = 0; k < kConvK; ++k) wk[i][k] = works ? F::load(w + (e + W * i) * kConvK + k, kConvK) : F::splat(0.f);
  }
  for (int box = blockIdx.y; box < boxes; box += gridDim.y) {
    const int t0 = box * kTcRows + warp * kMine, t1 = min(t0 + kMine, seqs.rows);
    if (!mbar_wait(&full[stage], round)) { atomicExch(&g_conv_status, MB200_DEV_WAIT_TIMEOUT); return; }
    // row t of the box's; channel of this lane
    const T* const in = reinterpret_cast<const T*>(smem + stage * kBytes) + (warp * kMine + kConvK - 1) * kTcChannels + lane * V;
    auto at_row = [&](int i) { return *reinterpret_cast<const CVec<T, V>*>(in + i * kTcChannels); };
    const uint64_t firsts = s_firsts[stage] >> (warp * kMine);             // bit i: row t0 - 2 + i
    const Begins* const begins = s_begins[stage] + warp * kMine;
    auto enter = [&](int i) {                             // the three rows in front of row i
#pragma unroll
      for (int k = 0; k < kConvK - 1; ++k) {
        F xv[P];
        unpack<T, V, W>(at_row(i + k - (kConvK - 1)), xv);
#pragma unroll
        for (int j = 0; j < P; ++j) win[j][k] = xv[j];
      }
    };
    auto row = [&](const CVec<T, V>& q) {
      F xn[P], o[P];
      unpack<T, V, W>(q, xn);
#pragma unroll
      for (int i = 0; i < P; ++i) {
        F acc = pfma(wk[i][0], win[i][0], bv[i]);
        acc = pfma(wk[i][1], win[i][1], acc);
        acc = pfma(wk[i][2], win[i][2], acc);
        acc = pfma(wk[i][3], xn[i], acc);
        win[i][0] = win[i][1]; win[i][1] = win[i][2]; win[i][2] = xn[i];
        o[i] = pmul(acc, psigmoid(acc));
      }
      return pack<T, V, W>(o);
    };
    T* yp = y + int64_t(t0) * y_sl + e;
    if (works && t0 + kMine <= tail && (firsts & ((uint64_t(1) << (kBefore + kMine)) - 1)) == 0) {
      enter(0);
#pragma unroll
      for (int j = 0; j < kMine; ++j) cstore<T, V>(yp + j * y_sl, row(at_row(j)));
    } else if (works && t0 < seqs.rows) {
      // as above: rows lo to hi are this warp's, and what begins among its 8 leaves its window here
      auto first_at = [&](int i) { return (firsts >> (i + kBefore) & 1) != 0; };
      const int n = t1 - t0, last = max(0, min(n, tail - t0));
      int lo = 0, hi = last;
      constexpr int kFar = -2 * kConvK;
      const int in_front = first_at(-1) ? -1 : first_at(-2) ? -2 : kFar;
      const int at_end = n != kMine ? kFar : first_at(n - 1) ? n - 1 : first_at(n - 2) ? n - 2 : kFar;
      while (lo < n && lo - in_front < kConvK - 1 && !first_at(lo)) ++lo;
      while (t0 + hi < tail && hi - at_end < kConvK - 1 && !first_at(hi)) ++hi;
      enter(lo);
#pragma unroll 1
      for (int i = lo; i < hi; ++i) {
        if (first_at(i)) {
          const Begins q = begins[i + kBefore];
          if (q.slot >= 0 && q.old) {
            load_window<T, V, W>(windows + (q.slot * ED + e) * (kConvK - 1), win);
          } else {
#pragma unroll
            for (int j = 0; j < P; ++j)
#pragma unroll
              for (int k = 0; k < kConvK - 1; ++k) win[j][k] = F::splat(0.f);
          }
        }
        cstore<T, V>(yp + i * y_sl, row(at_row(i)));
      }
      CVec<T, V> zero;
#pragma unroll
      for (int i = 0; i < V; ++i) zero.v[i] = Elem<T>::from_f(0.f);
      for (int i = last; i < n; ++i) cstore<T, V>(yp + i * y_sl, zero);
      if (windows) {
        for (uint64_t own = firsts >> kBefore & ((uint64_t(1) << kMine) - 1); own; own &= own - 1) {
          const int i = __ffsll(int64_t(own)) - 1;
          const Begins q = begins[i + kBefore];
          if (q.slot >= 0) leave_window<T, V>(seqs, q.seq, t0 + i, q.old, x + e, x_sl, windows + (q.slot * ED + e) * (kConvK - 1));
        }
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty[stage]);
    next();
  }
}

// dx[t] = sum_j w[3-j] * dpre[t+j] over the rows t+j of t's sequence;  dw[k] = sum_t dpre[t] * in(t-3+k);  dbias = sum dpre;
// dpre[t] = dy[t] * silu'(pre[t]), pre recomputed from x.  Sequences that resume have no backward, so in = 0 before a first row.
// As on rectangles the windows hold as many rows as a group, dx trails by three rows, and the 4 warps of a CTA add their sums in shared memory.
// Of large tensors a thread takes 8 bytes of channels, and rows come through a ring in shared memory, groups ahead of the arithmetic: each thread copies
// what it reads itself, so its own waits are all it takes, and no register holds what is on its way.  16000 x 1536 without / with the ring: float32
// 70 (four channels) / 52 us (two; four 57), bfloat16 51 / 38 (two channels: 45).  Four stages of the ring take the L1 that the copies pass through
// (float32 62), two cost bfloat16 2 us.  Then bfloat16 waits for issue slots (half of them, with 13 warps an SM), float32 for HBM (5.6 TB/s).
constexpr int kPkBwdThreads = 128, kPkBwdWarps = kPkBwdThreads / 32, kPkBwdChunkMost = 128;
constexpr int kPkBwdStages = 3;                          // groups of four rows of x and dy
template <typename T, int V> constexpr int kPkBwdRing = V == 1 ? 0 : kPkBwdThreads * kPkBwdStages * 2 * kConvK * int(sizeof(T)) * V;
template <int V> constexpr int kPkBwdResident = V == 2 ? 5 : 4;

// This thread's copy of kBytes to shared memory; zeros if not `ok`.
template <int kBytes>
__device__ __forceinline__ void copy_ahead(void* to, const void* from, const void* valid, bool ok) {
  const unsigned at = unsigned(__cvta_generic_to_shared(to));
  const int n = ok ? kBytes : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(at), "l"(ok ? from : valid), "n"(kBytes), "r"(n) : "memory");
}

template <typename T, int V>
__global__ void __launch_bounds__(kPkBwdThreads, kPkBwdResident<V>)
conv1d_silu_packed_bwd_kernel(const Packed seqs, const T* __restrict__ x, const float* __restrict__ w, const float* __restrict__ bias,
                              const T* __restrict__ dy, T* __restrict__ dx, float* __restrict__ dw, float* __restrict__ dbias, int64_t ED,
                              int64_t x_sl, int64_t dy_sl, int64_t dx_sl, int chunk) {
  constexpr int kG = kConvK, kH = kConvK - 1, kStages = kPkBwdStages;
  constexpr bool kRing = V > 1;
  extern __shared__ __align__(16) unsigned char ring[];
  constexpr int kBits = kH + kPkBwdWarps * kPkBwdChunkMost + kH;
  __shared__ float s_acc[32 * V * (kConvK + 1)];          // per channel of the CTA: dw[0..3], dbias
  __shared__ unsigned s_first[(kBits + 31) / 32 + 1];     // bit i: a sequence begins at row T0 - 3 + i
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int T0 = int(blockIdx.x) * kPkBwdWarps * chunk;
  for (int i = threadIdx.x; i < 32 * V * (kConvK + 1); i += kPkBwdThreads) s_acc[i] = 0.f;
  for (int i = threadIdx.x; i < (kBits + 31) / 32 + 1; i += kPkBwdThreads) s_first[i] = 0;
  __syncthreads();
  const int tail = seqs.start(seqs.sequences);
  for (int r = threadIdx.x; r <= seqs.sequences; r += kPkBwdThreads) {
    const int at = seqs.start(r) - (T0 - kH);
    if (at >= 0 && at < kBits) atomicOr(&s_first[at >> 5], 1u << (at & 31));
  }
  __syncthreads();
  const int64_t e = (int64_t(blockIdx.y) * 32 + lane) * V;
  const int t0 = T0 + warp * chunk, t1 = min(seqs.rows, t0 + chunk);
  if (e < ED && t0 < seqs.rows) {
    constexpr int W = (V % 2 == 0) ? 2 : 1, P = V / W;
    using F = Pk<W>;
    F wk[P][kConvK], bv[P];
#pragma unroll
    for (int i = 0; i < P; ++i) {
      bv[i] = bias ? F::load(bias + e + W * i, 1) : F::splat(0.f);
#pragma unroll
      for (int k = 0; k < kConvK; ++k) wk[i][k] = F::load(w + (e + W * i) * kConvK + k, kConvK);
    }
    F xw[P][kG], dw_[P][kG], dwacc[P][kConvK], dbacc[P];
#pragma unroll
    for (int i = 0; i < P; ++i) {
      dbacc[i] = F::splat(0.f);
#pragma unroll
      for (int k = 0; k < kConvK; ++k) dwacc[i][k] = F::splat(0.f);
#pragma unroll
      for (int k = 0; k < kG; ++k) dw_[i][k] = F::splat(0.f);
    }
    const Firsts firsts{s_first, T0 - kH};
    auto firsts_at = [&](int t) { return firsts.from(t - kH) & 0x7fu; };       // of rows t - 3 .. t + 3
    const T* xg = x + int64_t(t0) * x_sl + e;
    const T* gg = dy + int64_t(t0) * dy_sl + e;
    T* og = dx + int64_t(t0 - kH) * dx_sl + e;
    {
      const unsigned f = firsts_at(t0) & 7u;              // of t0-3 .. t0-1: what lies before the last of them is not in the sequence
#pragma unroll
      for (int k = 0; k < kH; ++k) {
        F xv[P];
        unpack<T, V, W>(cload<T, V>(xg + (k - kH) * x_sl, t0 + k >= kH && t0 + k - kH < tail && (f >> (k + 1)) == 0), xv);
#pragma unroll
        for (int i = 0; i < P; ++i) xw[i][k + 1] = xv[i];
      }
    }
    const F one = F::splat(1.f), mone = F::splat(-1.f), zero = F::splat(0.f);
    const int own = max(0, min(t1, tail) - t0), end = min(tail, t1 + kH) - t0;
    CVec<T, V>* const mine = reinterpret_cast<CVec<T, V>*>(ring) + warp * (kStages * 2 * kG * 32) + lane;
    int stage = 0;
    auto ahead = [&](int s0, int to) {
      if (s0 < own + kH) {
#pragma unroll
        for (int j = 0; j < kG; ++j) {
          copy_ahead<sizeof(T) * V>(mine + (to * 2 * kG + j) * 32, xg, x, s0 + j < end);
          copy_ahead<sizeof(T) * V>(mine + (to * 2 * kG + kG + j) * 32, gg, x, s0 + j < end);
          xg += x_sl; gg += dy_sl;
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto group = [&](auto plain, int s0, unsigned f) {    // f: bits of rows s0 - 3 .. s0 + 3; plain: inside the chunk, and none set
      constexpr bool kPlain = decltype(plain)::value;
      CVec<T, V> qx[kG], qg[kG];
#pragma unroll
      for (int j = 0; j < kG; ++j) {
        if constexpr (kRing) {
          qx[j] = mine[(stage * 2 * kG + j) * 32];
          qg[j] = mine[(stage * 2 * kG + kG + j) * 32];
        } else {
          qx[j] = cload<T, V>(xg, kPlain || s0 + j < end);
          qg[j] = cload<T, V>(gg, kPlain || s0 + j < end);
          xg += x_sl; gg += dy_sl;
        }
      }
#pragma unroll
      for (int j = 0; j < kG; ++j) {
        F g[P], xn[P], o[P];
        unpack<T, V, W>(qg[j], g);
        unpack<T, V, W>(qx[j], xn);
        const bool fresh = !kPlain && (f >> (kH + j) & 1);
        // how many rows behind t-3 its dx takes in: up to the first row of the next sequence
        const int reach = kPlain ? 3 : f >> (j + 1) & 1 ? 0 : f >> (j + 2) & 1 ? 1 : f >> (j + 3) & 1 ? 2 : 3;
#pragma unroll
        for (int i = 0; i < P; ++i) {
          if (fresh) {
#pragma unroll
            for (int k = 0; k < kG; ++k) xw[i][k] = zero;
          }
          xw[i][j] = xn[i];
          F pre = bv[i];
#pragma unroll
          for (int k = 0; k < kConvK; ++k) pre = pfma(wk[i][k], xw[i][(j + 1 + k) % kG], pre);
          const F sg = psigmoid(pre);
          const F dp = pmul(pmul(g[i], sg), pfma(pre, pfma(sg, mone, one), one));
          dw_[i][j] = dp;
          // dx[t-3] = w3*dpre[t-3] + w2*dpre[t-2] + w1*dpre[t-1] + w0*dpre[t]
          F acc = pmul(wk[i][kH], dw_[i][(j + 1) % kG]);
#pragma unroll
          for (int k = 1; k < kConvK; ++k)
            if (kPlain || k <= reach) acc = pfma(wk[i][kH - k], dw_[i][(j + 1 + k) % kG], acc);
          o[i] = acc;
          if (kPlain || s0 + j < own) {
            dbacc[i] = padd(dbacc[i], dp);
#pragma unroll
            for (int k = 0; k < kConvK; ++k) dwacc[i][k] = pfma(dp, xw[i][(j + 1 + k) % kG], dwacc[i][k]);
          }
        }
        if (kPlain || (s0 + j >= kH && s0 + j - kH < own)) cstore<T, V>(og, pack<T, V, W>(o));
        og += dx_sl;
      }
    };
    if constexpr (kRing) {
#pragma unroll
      for (int i = 0; i < kStages - 1; ++i) ahead(i * kG, i);
    }
#pragma unroll 1
    for (int s0 = 0; s0 < own + kH; s0 += kG) {
      if constexpr (kRing) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
        ahead(s0 + (kStages - 1) * kG, stage == 0 ? kStages - 1 : stage - 1);
      }
      const unsigned f = firsts_at(t0 + s0);
      if (f == 0 && s0 >= kH && s0 + kG <= own && s0 + kG <= end) group(std::true_type{}, s0, f);
      else group(std::false_type{}, s0, f);
      if (kRing && ++stage == kStages) stage = 0;
    }
    CVec<T, V> none;                                      // rows of no sequence, whatever the filter holds
#pragma unroll
    for (int i = 0; i < V; ++i) none.v[i] = Elem<T>::from_f(0.f);
    for (int t = max(t0, tail); t < t1; ++t) cstore<T, V>(dx + int64_t(t) * dx_sl + e, none);
#pragma unroll
    for (int i = 0; i < P; ++i) {
#pragma unroll
      for (int u = 0; u < W; ++u) {
        float* a = s_acc + (lane * V + i * W + u) * (kConvK + 1);
#pragma unroll
        for (int k = 0; k < kConvK; ++k) {
          float val;
          if constexpr (W == 1) val = dwacc[i][k].v; else val = u ? dwacc[i][k].v.y : dwacc[i][k].v.x;
          atomicAdd(a + k, val);
        }
        float dbv;
        if constexpr (W == 1) dbv = dbacc[i].v; else dbv = u ? dbacc[i].v.y : dbacc[i].v.x;
        atomicAdd(a + kConvK, dbv);
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 32 * V * (kConvK + 1); i += kPkBwdThreads) {
    const int64_t ch = int64_t(blockIdx.y) * 32 * V + i / (kConvK + 1);
    const int k = i % (kConvK + 1);
    if (ch >= ED) continue;
    if (k < kConvK) atomicAdd(dw + ch * kConvK + k, s_acc[i]);
    else if (dbias) atomicAdd(dbias + ch, s_acc[i]);
  }
}

// Rows of a warp, a multiple of `unit`: as many as make the rounds of CTAs that fit the SMs, and what each round costs besides its rows (`extra` rows'
// worth: the way of the first loads, the filter, where sequences begin, the rows in front), cheapest.
int packed_chunk(int64_t rows, int64_t cols, int warps, int resident, int unit, int most, int extra) {
  int best = unit;
  int64_t best_cost = int64_t(1) << 62;
  for (int c = unit; c <= most; c += unit) {
    const int64_t ctas = cols * ((rows + warps * c - 1) / (warps * c)), fit = int64_t(sm_count()) * resident;
    const int64_t cost = (ctas + fit - 1) / fit * (c + extra);
    if (cost < best_cost) { best_cost = cost; best = c; }
  }
  return best;
}

// Channels of a thread of the backward: 8 bytes of them save instructions, one gives more warps.  us so / with one, kernels in a graph:
//            1000 x 512   3000 x 1000   8000 x 512   4000 x 1536   2000 x 5120   8000 x 1536   16000 x 1536
// float32     5.2 / 4.7     9.9 / 9.2    11.4 / 11.8  16.0 / 21.5   24.6 / 40.9   29.7 / 49.3   53.5 / 90.5
// bfloat16    6.3 / 4.8    11.6 / 10.3   13.9 / 11.4  16.6 / 15.9   22.1 / 35.3   24.8 / 43.7   38.0 / 84.7
bool one_channel(int64_t values, int dtype) { return values <= (dtype == MB200_F32 ? int64_t(9) << 19 : int64_t(7) << 20); }

int check_conv(const mb200_packed* seqs, int64_t ED, int K, int dtype) {
  if (const int rc = packed_check(seqs)) return rc;
  if (ED < 0) return MB200_EINVAL;
  if (K != kConvK || ED > int64_t(65535) * 32) return MB200_ETOOBIG;
  return dtype != MB200_F32 && dtype != MB200_BF16 ? MB200_EDTYPE : MB200_OK;
}

}  // namespace
}  // namespace mb200

using namespace mb200;

// Reads (and clears) the device-side status word of the packed convolution.  Synchronises the device.
int mb200_conv_device_status() {
  int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_conv_status, sizeof(int)) != cudaSuccess) return -1;
  if (v) cudaMemcpyToSymbol(g_conv_status, &zero, sizeof(int));
  return v;
}

extern "C" int mb200_conv1d_silu_packed_fwd(const mb200_packed* seqs, const void* x, const float* w, const float* bias, void* windows, void* y,
                                            int64_t ED, int K, int64_t x_sl, int64_t y_sl, int dtype, void* stream) {
  if (const int rc = check_conv(seqs, ED, K, dtype)) return rc;
  if (seqs->rows == 0 || ED == 0) return MB200_OK;
  if (!x || !w || !y || (seqs->slots && !windows)) return MB200_EINVAL;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const Packed k = packed_of(*seqs, 0);
  if (!seqs->slots) windows = nullptr;
  const bool bf = dtype == MB200_BF16;
  const int channels = kTcBytes / (bf ? 2 : 4);
  CUtensorMap map;
  if (conv_vec_ok(ED, channels / 32, {x, y, (const void*)windows}, {y_sl}) && tma_compatible(x, 0, x_sl, ED, bf ? 2 : 4, channels) &&
      tma_encode(&map, x, bf, 1, seqs->rows, ED, 0, x_sl, channels, kTcBox)) {
    const int64_t across = (ED + channels - 1) / channels, boxes = (seqs->rows + kTcRows - 1) / kTcRows;
    const int64_t down = int64_t(sm_count()) * kTcResident / across;
    const dim3 walk(unsigned(across), unsigned(down < 1 ? 1 : min64(down, boxes)));
#define MB200_CONV_FWD(TT) \
  conv1d_silu_packed_tma_kernel<TT><<<walk, kTcThreads, kTcStages * kTcBox * kTcBytes, st>>>(map, k, (const TT*)x, w, bias, (TT*)y, (TT*)windows, ED, x_sl, y_sl)
    if (bf) MB200_CONV_FWD(__nv_bfloat16); else MB200_CONV_FWD(float);
#undef MB200_CONV_FWD
    return check_launch();
  }
  const int64_t cols = (ED + 31) / 32;
  const int chunks = packed_chunk(seqs->rows, cols, kPkWarps, kPkResident, kPkChunk, 16 * kPkChunk, 16) / kPkChunk;
  const dim3 grid(unsigned((seqs->rows + kPkWarps * kPkChunk * chunks - 1) / (kPkWarps * kPkChunk * chunks)), unsigned(cols));
#define MB200_CONV_FWD(TT) \
  conv1d_silu_packed_fwd_kernel<TT><<<grid, kPkThreads, 0, st>>>(k, (const TT*)x, w, bias, (TT*)y, (TT*)windows, ED, x_sl, y_sl, chunks)
  if (bf) MB200_CONV_FWD(__nv_bfloat16); else MB200_CONV_FWD(float);
#undef MB200_CONV_FWD
  return check_launch();
}

extern "C" int mb200_conv1d_silu_packed_bwd(const mb200_packed* seqs, const void* x, const float* w, const float* bias, const void* dy,
                                            void* dx, float* dw, float* dbias, int64_t ED, int K, int64_t x_sl, int64_t dy_sl,
                                            int64_t dx_sl, int dtype, void* stream) {
  if (const int rc = check_conv(seqs, ED, K, dtype)) return rc;
  if (seqs->rows == 0 || ED == 0) return MB200_OK;
  if (!x || !w || !dy || !dx || !dw || seqs->slots) return MB200_EINVAL;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int kv = dtype == MB200_F32 ? 2 : 4;
  const bool vec = !one_channel(seqs->rows * ED, dtype) && conv_vec_ok(ED, kv, {x, dy, (const void*)dx}, {x_sl, dy_sl, dx_sl});
  const int v = vec ? kv : 1;
  const int64_t cols = (ED + 32 * int64_t(v) - 1) / (32 * int64_t(v));
  const int chunk = packed_chunk(seqs->rows, cols, kPkBwdWarps, v == 2 ? kPkBwdResident<2> : kPkBwdResident<1>, 8, kPkBwdChunkMost, 16);
  const dim3 grid(unsigned((seqs->rows + kPkBwdWarps * chunk - 1) / (kPkBwdWarps * chunk)), unsigned(cols));
  const Packed k = packed_of(*seqs, 0);
#define MB200_CONV_BWD(TT, VV)                                                                                                                  \
  {                                                                                                                                             \
    auto* const kernel = conv1d_silu_packed_bwd_kernel<TT, VV>;                                                                                 \
    constexpr int bytes = kPkBwdRing<TT, VV>;                                                                                                   \
    if (bytes && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return MB200_ELAUNCH;         \
    kernel<<<grid, kPkBwdThreads, bytes, st>>>(k, (const TT*)x, w, bias, (const TT*)dy, (TT*)dx, dw, dbias, ED, x_sl, dy_sl, dx_sl, chunk);     \
  }
  if (dtype == MB200_F32) { if (vec) MB200_CONV_BWD(float, 2) else MB200_CONV_BWD(float, 1) }
  else { if (vec) MB200_CONV_BWD(__nv_bfloat16, 4) else MB200_CONV_BWD(__nv_bfloat16, 1) }
#undef MB200_CONV_BWD
  return check_launch();
}
