// Sequences of different lengths laid end to end: sequence r is the rows cu[r] .. cu[r+1] - 1 of (rows, channels) tensors, and what
// belongs to a sequence (its state, its convolution window) lies in a slot of a pool.
#pragma once
#include "common.cuh"

namespace mb200 {

// `cu` is data on the device that the host has not seen: whatever it holds, no row outside [0, rows) is touched.  A slot outside
// the pool means that the sequence has none: it starts from nothing and leaves nothing.
struct Packed {
  const int32_t* cu = nullptr;
  const int64_t* slots = nullptr;
  const uint8_t* resume = nullptr;
  int sequences = 0, rows = 0;
  int piece = 0;                           // a sequence is cut at every `piece` rows (a multiple of 16; 0: not at all)
  int parts = 1;                           // carries are computed for parts of a piece, so many of them (each a multiple of 16 rows)
  int64_t n_slots = 0;

  __device__ __forceinline__ int start(int r) const {
    return r <= 0 ? 0 : min(max(__ldg(cu + r), 0), rows);
  }
  // The rows behind the last sequence are number `sequences`.
  __device__ __forceinline__ int end(int r, int begin) const { return r < sequences ? max(begin, start(r + 1)) : rows; }
  __device__ __forceinline__ int64_t slot(int r) const {
    if (!slots || r >= sequences) return -1;
    const int64_t s = __ldg(slots + r);
    return s >= 0 && s < n_slots ? s : -1;
  }
  __device__ __forceinline__ bool resumes(int r) const { return resume && __ldg(resume + r) != 0; }
};

// How many pieces a launch has to cover when only the number of rows and of sequences is known: sequence r's are numbered from
// cu[r] / piece + r on, which leaves room for all of them (the rows behind the last sequence are cut likewise) and needs no
// sums over lengths; numbers nothing uses are empty.
inline int64_t packed_items(int64_t rows, int64_t sequences, int64_t piece) { return (piece ? rows / piece : 0) + sequences + 1; }
// Saved states likewise: sequence r's chunk c is entry cu[r] / kChunk + r + c.
inline int64_t packed_chunks(int64_t rows, int64_t sequences, int chunk) { return rows / chunk + sequences; }

struct PackedItem {
  int seq;
  int begin, end;                          // its rows
  int pc, pieces;                          // which of its pieces (of its parts, in a carry pass), and how many pieces it has
  int lo, hi;                              // the rows of that; lo == hi: none
  int first_part, n_parts;                 // its parts: the number of the first, how many
};

// What a launch goes through: the pieces; the parts whose carry something to the right needs (those in front of the last piece, or all but the last
// part, whose decay products a backward needs); those whose carry something to the left needs (all behind the first piece).
enum PackedPass { kPieces, kPartsBefore, kPartsButLast, kPartsBehind };

// The item that CTA row `nth` of a grid takes, called by all NT threads of the CTA.  With up to NT sequences, each a thread's, whole
// pieces come first and the others after them by their length, longest first: CTAs start in that order, and what starts last decides how long the
// SMs wait for the last one.  Two scans over the threads in shared memory, next to the hundred microseconds of the pieces.
// More sequences than that are short ones for any number of rows, and taken as they come: a count of those numbered no higher finds
// the sequence in a round of loads for every NT of them.
template <int NT>
__device__ __forceinline__ PackedItem packed_item(const Packed& k, int nth, int tid, PackedPass pass = kPieces) {
  const int part = k.piece / k.parts, unit = pass == kPieces ? k.piece : part;
  // items of a sequence of n rows: `whole` of `unit` rows from number `from` on, and one of `rest` behind those
  auto items = [&](int n, int& from, int& whole, int& rest) {
    from = whole = 0;
    rest = n;
    if (!k.piece) return;
    whole = n / unit;
    rest = n - whole * unit;
    if (pass == kPieces) return;
    const int pieces = (n + k.piece - 1) / k.piece, parts = whole + (rest > 0);
    if (pieces < 2) {
      whole = rest = 0;
    } else if (pass == kPartsBehind) {
      from = k.parts;
      whole -= from;
    } else {
      whole = pass == kPartsBefore ? (pieces - 1) * k.parts : parts - 1;
      rest = 0;
    }
  };
  PackedItem r;
  r.seq = k.sequences;
  r.pc = 0;
  if (k.sequences <= NT) {
    __shared__ int s_at[2], s_whole[NT / 32 + 1];
    __shared__ int s_rest[NT];
    int from = 0, whole = 0, rest = 0;
    if (tid < k.sequences) {
      const int begin = k.start(tid);
      items(k.end(tid, begin) - begin, from, whole, rest);
    }
    s_rest[tid] = rest;
    if (tid == 0) s_at[0] = -1;
    int upto = whole;
    const int lane = tid & 31;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const int more = __shfl_up_sync(0xffffffffu, upto, s);
      if (lane >= s) upto += more;
    }
    if (lane == 31) s_whole[tid >> 5] = upto;
    __syncthreads();
    int all = 0;
#pragma unroll
    for (int w = 0; w < NT / 32; ++w) {
      if (w < tid >> 5) upto += s_whole[w];
      all += s_whole[w];
    }
    if (nth < all) {
      if (nth < upto && nth >= upto - whole) {
        s_at[0] = tid;
        s_at[1] = from + nth - (upto - whole);
      }
    } else if (rest) {
      int longer = 0;
      for (int q = 0; q < k.sequences; ++q) longer += s_rest[q] > rest || (s_rest[q] == rest && q < tid);
      if (longer == nth - all) {
        s_at[0] = tid;
        s_at[1] = from + whole;
      }
    }
    const int rests = __syncthreads_count(rest != 0);
    if (s_at[0] >= 0) {
      r.seq = s_at[0];
      r.pc = s_at[1];
    } else {
      r.pc = nth - all - rests;
    }
  } else {
    r.seq = nth;
    if (k.piece) {
      int below = 0;
      for (int base = 0; base <= k.sequences; base += NT) {
        const int q = base + tid;
        below += __syncthreads_count(q <= k.sequences && k.start(q) / unit + q <= nth);
      }
      r.seq = below - 1;
      r.pc = nth - (k.start(r.seq) / unit + r.seq);
    }
  }
  r.begin = k.start(r.seq);
  r.end = k.end(r.seq, r.begin);
  const int n = r.end - r.begin;
  r.pieces = k.piece ? (n + k.piece - 1) / k.piece : n > 0;
  r.n_parts = k.piece ? (n + part - 1) / part : 0;
  r.first_part = k.piece ? r.begin / part + r.seq : 0;
  r.lo = r.hi = r.begin;
  int from, whole, rest;
  items(n, from, whole, rest);
  if (pass != kPieces && r.seq == k.sequences) whole = rest = 0;
  if (r.pc >= from && r.pc < from + whole + (rest > 0)) {
    r.lo = r.begin + r.pc * unit;
    r.hi = r.pc < from + whole ? r.lo + unit : r.end;
  }
  return r;
}

// Columns [0, cols) of rows [lo, hi) become zero; `p` points at row 0.
template <typename T, int NT>
__device__ __forceinline__ void zero_rows(T* p, int64_t stride, int lo, int hi, int cols, int tid) {
  if (!p) return;
  for (int64_t i = tid; i < int64_t(hi - lo) * cols; i += NT) p[(lo + i / cols) * stride + i % cols] = Elem<T>::from_f(0.f);
}

inline Packed packed_of(const mb200_packed& s, int64_t piece, int64_t parts = 1) {
  Packed k;
  k.cu = s.cu_seqlens; k.slots = s.slots; k.resume = s.resume; k.n_slots = s.n_slots;
  k.sequences = int(s.sequences); k.rows = int(s.rows); k.piece = int(piece); k.parts = int(parts);
  return k;
}
inline int packed_check(const mb200_packed* s) {
  if (!s || s->sequences < 0 || s->rows < 0 || s->n_slots < 0) return MB200_EINVAL;
  if (s->sequences > 0 && !s->cu_seqlens) return MB200_EINVAL;
  if (s->rows >= (int64_t(1) << 30) || s->sequences > 65534) return MB200_ETOOBIG;
  return MB200_OK;
}

}  // namespace mb200
