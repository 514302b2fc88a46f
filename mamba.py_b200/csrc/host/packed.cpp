// Sequences of different lengths laid end to end, with their states in slots of a pool: scan and convolution; and beams on those slots.
#include <algorithm>
#include <cmath>
#include "host.h"

namespace mb200_host {
void same_device(const Tensor& on, std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    TORCH_CHECK(!t->defined() || t->device() == on.device(), "mamba_b200: tensors on ", on.device(), " and ", t->device(), " in one call");
}

Tensor as_type(const Tensor& t, at::ScalarType dt, const char* what) {
  if (!t.defined()) return t;
  const auto d = t.scalar_type();
  const bool ok = dt == at::kBool ? d == at::kBool : d == at::kInt || d == at::kLong;
  TORCH_CHECK_TYPE(ok, "mamba_b200: ", what, dt == at::kBool ? " should be bool, got " : " should be int32 or int64, got ", d);
  return (d == dt ? t : t.to(dt)).contiguous();
}

// A pool is written where it lies.
void check_pool(const Tensor& pool, at::IntArrayRef entry, at::ScalarType dt, const char* what) {
  TORCH_CHECK(pool.dim() == int64_t(entry.size()) + 1 && pool.sizes().slice(1) == entry, "mamba_b200: ", what, " should be slots of ", entry,
              ", got ", pool.sizes());
  TORCH_CHECK_VALUE(pool.scalar_type() == dt && pool.is_contiguous(), "mamba_b200: ", what, " should be contiguous ", dt,
                    ", because they are updated in place");
  TORCH_CHECK(!pool.requires_grad(), "mamba_b200: ", what, " are updated in place and take no part in automatic differentiation");
}
void written(const Tensor& pool) {
  if (!pool.is_inference()) torch::autograd::impl::bump_version(pool);
}

namespace {

// The sequences of a call: cu_seqlens (R + 1), and for those that keep a state slots (R) and which of them resume.
struct Sequences {
  Tensor cu, slots, resume;
  int64_t rows = 0, n_slots = 0;
  Sequences() = default;
  Sequences(const Tensor& x, const Tensor& cu_, const Tensor& pool, const Tensor& slots_, const Tensor& resume_) {
    TORCH_CHECK(cu_.dim() == 1 && cu_.size(0) >= 1, "mamba_b200: cu_seqlens should have one dimension and an entry more than sequences, got ", cu_.sizes());
    TORCH_CHECK(pool.defined() == slots_.defined(), "mamba_b200: a pool and the slots in it come together");
    TORCH_CHECK(slots_.defined() || !resume_.defined(), "mamba_b200: a sequence resumes from its slot; there are no slots");
    same_device(x, {&cu_, &pool, &slots_, &resume_});
    rows = x.size(0);
    cu = as_type(cu_, at::kInt, "cu_seqlens");
    slots = as_type(slots_, at::kLong, "slots");
    resume = as_type(resume_, at::kBool, "resume");
    const int64_t n = cu.size(0) - 1;
    if (slots.defined()) shape_is(slots, {n}, "slots");
    if (resume.defined()) shape_is(resume, {n}, "resume");
    if (pool.defined()) n_slots = pool.size(0);
  }
  mb200_packed abi() const {
    return mb200_packed{static_cast<const int32_t*>(cu.data_ptr()), cu.size(0) - 1, rows, static_cast<const int64_t*>(ptr(slots)),
                        static_cast<const uint8_t*>(ptr(resume)), n_slots};
  }
  int64_t count() const { return cu.size(0) - 1; }
};

// A (rows, width) tensor as a tensor map can describe it.
bool on_grid(const Tensor& t) {
  return !t.defined() || (reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && t.stride(0) * t.element_size() % 16 == 0 && t.stride(0) >= t.size(1));
}

struct PackedScan {
  Tensor x, delta, A, B, C, D, z, bias;
  Sequences seqs;
  int64_t piece_len = 0, parts = 1;
  int flags() const { return (bias.defined() ? MB200_DELTA_SOFTPLUS : 0) | MB200_PAIRED_STATES; }
  int code() const { return dtype_code(x.scalar_type()); }
  int64_t rows() const { return x.size(0); }
  int64_t width() const { return x.size(1); }
  int64_t states() const { return A.size(1); }
  int64_t n_parts() const { return mb200_packed_parts(rows(), seqs.count(), piece_len / parts); }
  bool maps() const {
    return on_grid(x) && on_grid(delta) && on_grid(z) && on_grid(B) && on_grid(C) && width() * x.element_size() % 16 == 0;
  }
};

// Slices of x_proj's output are often off the 16-byte grid; they are copied onto it as for rectangles (scan.cpp).
void align_bc(PackedScan& a) {
  if (!(on_grid(a.x) && on_grid(a.delta) && on_grid(a.z)) || a.width() * a.x.element_size() % 16 || (on_grid(a.B) && on_grid(a.C))) return;
  const int64_t N = a.B.size(1), es = a.B.element_size();
  if (a.B.strides() == a.C.strides() && static_cast<char*>(a.C.data_ptr()) - static_cast<char*>(a.B.data_ptr()) == N * es && a.B.stride(0) >= 2 * N) {
    const Tensor bc = strided(a.B, 0, {a.B.size(0), 2 * N}, a.B.strides()).contiguous();
    a.B = columns(bc, 0, N);
    a.C = columns(bc, N, N);
  } else {
    a.B = a.B.clone(at::MemoryFormat::Contiguous);
    a.C = a.C.clone(at::MemoryFormat::Contiguous);
  }
}

enum { kX, kDelta, kA, kB, kC, kD, kZ, kBias, kInputs };

struct PackedScanBackward : public torch::autograd::Node {
  Saved x, delta, A, B, C, D, z, bias, cu, carries, pieces;
  at::ScalarType types[kInputs];
  bool given[kInputs];
  int64_t piece_len = 0, parts = 1;
  std::vector<int64_t> D_shape, bias_shape;

  std::string name() const override { return "PackedSelectiveScanBackward"; }
  void release_variables() override {
    for (Saved* s : {&x, &delta, &A, &B, &C, &D, &z, &bias, &cu, &carries, &pieces}) s->reset();
  }
  variable_list apply(variable_list&& grads) override {
    variable_list out(kInputs);
    if (!grads[0].defined()) return out;
    const BelowAutograd guard_ad;
    PackedScan a{x.get(), delta.get(), A.get(), B.get(), C.get(), D.get(), z.get(), bias.get()};
    a.seqs.cu = cu.get();
    a.seqs.rows = a.rows();
    a.piece_len = piece_len;
    a.parts = parts;
    const c10::cuda::CUDAGuard guard(a.x.device());
    const auto dt = a.x.scalar_type();
    Tensor dy = rows(grads[0], dt);
    if (!on_grid(dy)) dy = dy.clone(at::MemoryFormat::Contiguous);          // (a contiguous one may begin off the grid)
    const int64_t T = a.rows(), W = a.width(), N = a.states();
    const Tensor dx = empty({T, W}, dt, a.x), dd = empty({T, W}, dt, a.x), dz = a.z.defined() ? empty({T, W}, dt, a.x) : Tensor();
    const Tensor acc = empty({2 * T * N + W * N + 2 * W}, at::kFloat, a.x);
    zero_fill(acc);
    const Tensor dB = alias(acc, 0, {T, N}), dC = alias(acc, T * N, {T, N}), dA = alias(acc, 2 * T * N, {W, N}),
                 dD = alias(acc, 2 * T * N + W * N, given[kD] ? D_shape : std::vector<int64_t>{W}),
                 db = a.bias.defined() ? alias(acc, 2 * T * N + W * N + W, bias_shape) : Tensor();
    const Tensor pg = piece_len ? empty({a.n_parts(), W, N}, at::kFloat, a.x) : Tensor(), car = carries.get(), pcs = pieces.get();
    const mb200_packed s = a.seqs.abi();
    check(mb200_sscan_packed_bwd(&s, ptr(a.x), ptr(a.delta), ptr(a.z), fptr(a.A), ptr(a.B), ptr(a.C), fptr(a.D), fptr(a.bias), ptr(dy), fptr(car),
                                 fptr(pcs), fptr(pg), ptr(dx), ptr(dd), ptr(dz), fptr(dB), fptr(dC), fptr(dA), fptr(dD), fptr(db), W, int(N),
                                 st(a.x, 0), st(a.delta, 0), st(a.z, 0), st(a.B, 0), st(a.C, 0), st(dy, 0), st(dx, 0), st(dd, 0), st(dz, 0),
                                 piece_len, parts, a.code(), a.flags(), cuda_stream()),
          "mb200_sscan_packed_bwd");
    check_status("mb200_sscan_packed_bwd");
    const Tensor all[kInputs] = {dx, dd, dA, dB, dC, dD, dz, db};
    Convert conv;
    for (int i = 0; i < kInputs; ++i) {
      if (!given[i] || !all[i].defined() || !task_should_compute_output(i)) continue;
      out[i] = convertible(types[i]) ? conv.cast(all[i], types[i]) : like(all[i], types[i]);
    }
    conv.run();
    return out;
  }
};

// The filter of `width` channels, (width, d_conv).
Tensor filter(const Tensor& weight, int64_t width) {
  numel_is(weight, width * weight.size(-1), "the filter");
  return f32(weight).view({width, weight.size(-1)});
}

struct PackedConvBackward : public torch::autograd::Node {
  Saved x, w, b, cu;
  at::ScalarType tx, tw, tb;
  std::vector<int64_t> w_shape, b_shape;
  std::string name() const override { return "PackedCausalConv1dSiluBackward"; }
  void release_variables() override {
    for (Saved* s : {&x, &w, &b, &cu}) s->reset();
  }
  variable_list apply(variable_list&& grads) override {
    variable_list out(3);
    if (!grads[0].defined()) return out;
    const BelowAutograd guard_ad;
    const Tensor xs = x.get(), w32 = w.get(), b32 = b.get();
    const c10::cuda::CUDAGuard guard(xs.device());
    const Tensor dy = rows(grads[0], xs.scalar_type());
    const int64_t T = xs.size(0), W = xs.size(1), K = w32.size(1);
    const Tensor dx = empty({T, W}, xs.scalar_type(), xs), acc = empty({W * K + W}, at::kFloat, xs);
    zero_fill(acc);
    const Tensor dw = alias(acc, 0, w_shape), db = b32.defined() ? alias(acc, W * K, b_shape) : Tensor();
    Sequences q;
    q.cu = cu.get();
    q.rows = T;
    const mb200_packed s = q.abi();
    check(mb200_conv1d_silu_packed_bwd(&s, ptr(xs), fptr(w32), fptr(b32), ptr(dy), ptr(dx), fptr(dw), fptr(db), W, int(K), st(xs, 0), st(dy, 0),
                                       st(dx, 0), dtype_code(xs.scalar_type()), cuda_stream()),
          "mb200_conv1d_silu_packed_bwd");
    out[0] = like(dx, tx);
    out[1] = like(dw, tw);
    if (db.defined()) out[2] = like(db, tb);
    return out;
  }
};

}  // namespace

// Where to cut sequences (length 0: nowhere), and into how many parts a piece goes for the carry passes, from a model of the time of the passes, as
// pick_pieces has it for rows of one length and with its measured times for 2048 rows with 1 / 2 / 3 CTAs on every SM.  Lengths are known to the
// device alone: one sequence is taken to be `longest`, the others to share the rest evenly.  A pass takes the longer of
//   all its CTAs' rows at the rate of as many CTAs as there are on an SM;
//   its whole pieces in rounds, the others in the gaps (a tenth more of them than there are if others compete: the longest do not spread
//     over the SMs evenly then, six SMs of 148 had two while ten had none);
//   with few whole pieces: the others, and then what is left of the whole ones at the pace of an SM of their own.
// The parts are as many as give the carry passes three CTAs on every SM, four at most and 48 rows at least: those passes go through pieces of the cut
// sequences alone, and waited for few long ones.
// Over 60 cases (1 to 64 sequences, 325 to 16384 rows, 32 to 5120 channels, both types, training and serving) the cut picked takes 3.6 % longer than the
// best of 13 on average and 16 % at most; not cutting takes up to nine times as long (one sequence of 16384 x 256: 616 us for 70).  Parts took 16384 rows
// of 1536 in 20 documents from 870 to 793 us of training, one sequence of 14213 among others from 291 to 267 of reading.
struct Cut { int64_t length, parts; };
constexpr int64_t kShortestPart = 48, kMostParts = 4;

static int64_t parts_of(int64_t piece, double whole, double tiles, double sms) {
  int64_t parts = std::min<int64_t>(kMostParts, std::max<int64_t>(1, int64_t(std::ceil(3 * sms / std::max(1.0, whole * tiles)))));
  while (parts > 1 && (piece % (16 * parts) || piece / parts < kShortestPart)) --parts;
  return parts;
}

// `piece`: a length to be taken as it is, or -1.
static Cut pick_cut(int64_t rows, int64_t sequences, int64_t longest, int64_t width, bool grad, int64_t piece = -1) {
  constexpr double kFill = 20, kFwdSaving[] = {0, 82, 123, 174}, kFwd[] = {0, 79, 121, 170}, kBwd[] = {0, 279, 378, 538},
                   kFwdCarry[] = {0, 55, 87, 125}, kBwdCarry[] = {0, 62, 94, 135};
  if (rows <= 0 || sequences <= 0 || longest <= 0 || piece == 0) return {0, 1};
  const double sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount, tiles = double((width + 31) / 32);
  const double rest = sequences > 1 ? double(std::max<int64_t>(rows - longest, 0)) / double(sequences - 1) : 0;
  struct Group { double length, count; };
  auto pass = [&](const Group (&g)[4], const double (&t)[4]) {
    double most = 0, n = 0, full = 0, work = 0, full_work = 0;
    for (const Group& q : g) most = q.count > 0 ? std::max(most, q.length) : most;
    if (most <= 0) return 0.0;
    for (const Group& q : g) {
      if (q.length <= 0) continue;
      n += q.count * tiles;
      work += (q.length + kFill) * q.count * tiles;
      if (q.length > 0.9 * most) {
        full += q.count * tiles;
        full_work += (q.length + kFill) * q.count * tiles;
      }
    }
    auto step = [&](int c) { return t[c] / 2048; };
    const int c = int(std::min(3.0, std::max(1.0, std::ceil(n / sms)))), per_sm = int(std::ceil(full * (n > full ? 1.1 : 1.0) / sms));
    double us = std::max(n >= sms ? work / sms * step(c) / c : 0.0, (most + kFill) * (per_sm / 3 * step(3) + step(per_sm % 3)));
    if (full <= 2 * sms && n > full) {
      const double others = (work - full_work) / sms * step(3) / 3 / (1 - std::min(0.9, full / sms / 3));
      us = std::max(us, others + (most - others / step(3)) * step(1.2 * full <= sms ? 1 : 2));
    }
    return us;
  };
  Cut best{0, 1};
  double best_us = 0;
  for (const int64_t S : {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 24, 32, 48}) {
    int64_t P = piece > 0 ? piece : (longest + 16 * S - 1) / (16 * S) * 16;
    if (piece < 0 && P >= 2 * 64) P = (P + 63) / 64 * 64;               // (divisible into parts)
    if (piece < 0 && S > 1 && P < 64) break;
    Group main[4] = {}, carry[4] = {};
    int k = 1;
    double whole = 0;
    for (const Group& q : {Group{double(longest), 1}, Group{rest, double(sequences - 1)}}) {
      if (q.length <= 0 || q.count <= 0) continue;
      const double pieces = S > 1 || piece > 0 ? std::ceil(q.length / double(P)) : 1;
      whole += q.count * (pieces - 1);
      main[k++] = Group{q.length - (pieces - 1) * double(P), q.count};
    }
    const int64_t parts = parts_of(P, whole, tiles, sms);
    if (piece > 0) return {P, parts};
    if (S > 1 && mb200_packed_parts(rows, sequences, P / parts) > 65535) break;      // more than a launch has room for
    main[0] = Group{double(P), whole};
    carry[0] = Group{double(P) / double(parts), whole * double(parts)};
    double us = pass(main, grad ? kFwdSaving : kFwd) + (grad ? pass(main, kBwd) : 0);
    if (whole > 0) us += pass(carry, kFwdCarry) + (grad ? pass(carry, kBwdCarry) : 0) + (grad ? 16 : 7);
    if (whole > 0 && sequences > 2) us *= 1.1;                          // the others are not even, and more of them will be cut
    if (S == 1 || us < best_us) {
      best = S == 1 ? Cut{0, 1} : Cut{P, parts};
      best_us = us;
    }
    if (S == 1 && us < (grad ? 24 : 12)) break;                         // nothing to gain, and 1 us of the host's to lose
  }
  return best;
}

Tensor selective_scan_packed(const Tensor& x, const Tensor& delta, const Tensor& A, const Tensor& B, const Tensor& C, const OptTensor& D_,
                             const OptTensor& z_, const OptTensor& bias_, const Tensor& cu, const OptTensor& states_, const OptTensor& slots_,
                             const OptTensor& resume_, std::optional<int64_t> max_length, std::optional<int64_t> piece_length) {
  const Tensor &D = value(D_), &z = value(z_), &bias = value(bias_), &states = value(states_), &slots = value(slots_), &resume = value(resume_);
  require_cuda(x, delta, A, B, C, D, z, bias, cu, states, slots, resume);
  refuse_tangents(x, delta, A, B, C, D, z, bias);
  const c10::cuda::CUDAGuard guard(x.device());
  TORCH_CHECK(x.dim() == 2 && A.dim() == 2, "mamba_b200: packed sequences are (rows, channels) tensors, got ", x.sizes());
  same_device(x, {&delta, &A, &B, &C, &D, &z, &bias});
  const int64_t T = x.size(0), W = x.size(1), N = A.size(1);
  shape_is(delta, {T, W}, "delta");
  if (z.defined()) shape_is(z, {T, W}, "z");
  shape_is(A, {W, N}, "A");
  shape_is(B, {T, N}, "B");
  shape_is(C, {T, N}, "C");
  numel_is(D, W, "D");
  numel_is(bias, W, "delta_bias");
  const auto dt = act_dtype(x, delta, z, B, C);
  const bool grad = wants_grad(x, delta, A, B, C, D, z, bias);
  if (states.defined()) {
    check_pool(states, {W, N}, at::kFloat, "states");
    TORCH_CHECK(!grad, "mamba_b200: a scan that leaves its states in slots has no gradient; call it under torch.no_grad()");
  }
  TORCH_CHECK_VALUE(!max_length || *max_length >= 0, "mamba_b200: max_length should not be negative");
  TORCH_CHECK_VALUE(!piece_length || (*piece_length >= 0 && *piece_length % 16 == 0), "mamba_b200: piece_length should be a multiple of 16");
  PackedScan a;
  Tensor y, carries, pieces;
  {
    const BelowAutograd guard_ad;
    a = PackedScan{rows(x, dt), rows(delta, dt), f32(A), rows(B, dt), rows(C, dt), f32(D), rows(z, dt), f32(bias),
                   Sequences(x, cu, states, slots, resume)};
    align_bc(a);
    const int64_t R = a.seqs.count(), longest = std::min(T, max_length.value_or(T));
    if (N == 16 && a.maps() && (!piece_length || *piece_length < longest)) {
      const Cut cut = pick_cut(T, R, longest, W, grad, piece_length.value_or(-1));
      a.piece_len = cut.length < longest ? cut.length : 0;
      a.parts = a.piece_len ? cut.parts : 1;
    }
    y = empty({T, W}, dt, a.x);
    if (grad) carries = empty({mb200_packed_saved_states(T, R), W, N}, at::kFloat, a.x);
    if (a.piece_len) pieces = empty({2, a.n_parts(), W, N}, at::kFloat, a.x);
    const mb200_packed s = a.seqs.abi();
    check(mb200_sscan_packed_fwd(&s, ptr(a.x), ptr(a.delta), ptr(a.z), fptr(a.A), ptr(a.B), ptr(a.C), fptr(a.D), fptr(a.bias), fptr(states), ptr(y),
                                 fptr(carries), fptr(pieces), W, int(N), st(a.x, 0), st(a.delta, 0), st(a.z, 0), st(a.B, 0), st(a.C, 0), st(y, 0),
                                 a.piece_len, a.parts, a.code(), a.flags(), cuda_stream()),
          "mb200_sscan_packed_fwd");
    check_status("mb200_sscan_packed_fwd");
  }
  if (states.defined()) written(states);
  if (grad) {
    auto node = new_node<PackedScanBackward>();
    const Tensor* in[kInputs] = {&x, &delta, &A, &B, &C, &D, &z, &bias};
    for (int i = 0; i < kInputs; ++i) {
      node->given[i] = in[i]->defined();
      node->types[i] = type_of(*in[i]);
    }
    node->set_next_edges(torch::autograd::collect_next_edges(x, delta, A, B, C, D, z, bias));
    node->x.save(a.x); node->delta.save(a.delta); node->A.save(a.A); node->B.save(a.B); node->C.save(a.C); node->D.save(a.D);
    node->z.save(a.z); node->bias.save(a.bias); node->cu.save(a.seqs.cu); node->carries.save(carries); node->pieces.save(pieces);
    node->piece_len = a.piece_len; node->parts = a.parts;
    if (D.defined()) node->D_shape = D.sizes().vec();
    if (bias.defined()) node->bias_shape = bias.sizes().vec();
    torch::autograd::set_history(y, node);
  }
  return y;
}

Tensor conv1d_silu_packed(const Tensor& x, const Tensor& weight, const OptTensor& bias_, const Tensor& cu, const OptTensor& windows_,
                          const OptTensor& slots_, const OptTensor& resume_) {
  const Tensor &bias = value(bias_), &windows = value(windows_), &slots = value(slots_), &resume = value(resume_);
  require_cuda(x, weight, bias, cu, windows, slots, resume);
  refuse_tangents(x, weight, bias);
  const c10::cuda::CUDAGuard guard(x.device());
  TORCH_CHECK(x.dim() == 2, "mamba_b200: packed sequences are (rows, channels) tensors, got ", x.sizes());
  same_device(x, {&weight, &bias});
  const auto dt = act_dtype(x);
  const bool grad = wants_grad(x, weight, bias);
  const int64_t T = x.size(0), W = x.size(1), K = weight.size(-1);
  TORCH_CHECK(K == 4, "mamba_b200: the convolution of packed sequences takes filters of 4 taps (d_conv 4), got ", K);
  if (windows.defined()) {
    check_pool(windows, {W, K - 1}, dt, "windows");
    TORCH_CHECK(!grad, "mamba_b200: a convolution that leaves its windows in slots has no gradient; call it under torch.no_grad()");
  }
  Tensor y, xs, w32, b32;
  Sequences q;
  {
    const BelowAutograd guard_ad;
    xs = rows(x, dt);
    w32 = filter(weight, W);
    b32 = f32(bias);
    numel_is(b32, W, "the bias");
    q = Sequences(x, cu, windows, slots, resume);
    y = empty({T, W}, dt, xs);
    const mb200_packed s = q.abi();
    check(mb200_conv1d_silu_packed_fwd(&s, ptr(xs), fptr(w32), fptr(b32), ptr(windows), ptr(y), W, int(K), st(xs, 0), st(y, 0), dtype_code(dt),
                                       cuda_stream()),
          "mb200_conv1d_silu_packed_fwd");
    check_status("mb200_conv1d_silu_packed_fwd");
  }
  if (windows.defined()) written(windows);
  if (grad) {
    auto node = new_node<PackedConvBackward>();
    node->set_next_edges(torch::autograd::collect_next_edges(x, weight, bias));
    node->x.save(xs); node->w.save(w32); node->b.save(b32); node->cu.save(q.cu);
    node->tx = type_of(x); node->tw = type_of(weight); node->tb = type_of(bias);
    node->w_shape = weight.sizes().vec();
    if (bias.defined()) node->b_shape = bias.sizes().vec();
    torch::autograd::set_history(y, node);
  }
  return y;
}

// ------------------------------------------------------------------------------------------------------ beams

std::tuple<Tensor, Tensor, Tensor> beam_select(const Tensor& logits, const Tensor& scores, std::optional<int64_t> num_, const OptTensor& finished_,
                                               std::optional<int64_t> end_token) {
  const Tensor& finished = value(finished_);
  require_cuda(logits, scores, finished);
  same_device(logits, {&scores, &finished});
  const c10::cuda::CUDAGuard guard(logits.device());
  const BelowAutograd guard_ad;
  TORCH_CHECK(scores.dim() == 2, "mamba_b200: scores should be (groups, beams), got ", scores.sizes());
  const int64_t G = scores.size(0), B = scores.size(1);
  TORCH_CHECK(logits.dim() == 3 ? logits.size(0) == G && logits.size(1) == B : logits.dim() == 2 && logits.size(0) == G * B,
              "mamba_b200: logits should be (groups, beams, vocabulary) or (groups * beams, vocabulary) for scores of ", scores.sizes(), ", got ",
              logits.sizes());
  const int64_t V = logits.size(-1), num = num_.value_or(B);
  TORCH_CHECK(B >= 1 && V >= 1, "mamba_b200: there is nothing to select from");
  TORCH_CHECK_VALUE(num >= 1 && num <= B * V, "mamba_b200: num should be 1 to beams * vocabulary, got ", num);
  TORCH_CHECK_TYPE(scores.scalar_type() == at::kFloat, "mamba_b200: scores should be float32, got ", scores.scalar_type());
  if (finished.defined()) {
    shape_is(finished, {G, B}, "finished");
    TORCH_CHECK_VALUE(end_token && *end_token >= 0 && *end_token < V, "mamba_b200: finished beams need an end_token of the vocabulary");
  }
  const auto dt = act_dtype(logits);
  // rows of one stride
  Tensor rows_ = logits;
  if (logits.dim() == 3 && G > 1 && B > 1 && logits.stride(0) != B * logits.stride(1)) rows_ = logits.contiguous();
  if (rows_.stride(-1) != 1 && V > 1) rows_ = logits.contiguous();
  const int64_t stride = rows_.dim() == 2 ? rows_.stride(0) : B > 1 ? rows_.stride(1) : rows_.stride(0);
  const Tensor s = scores.contiguous(), f = as_type(finished, at::kBool, "finished");
  const Tensor out = empty({G, num}, at::kFloat, logits), tokens = empty({G, num}, at::kLong, logits), parents = empty({G, num}, at::kLong, logits);
  const int64_t bytes = num <= 64 ? mb200_beam_select_scratch_bytes(G, B, V, int(num)) : 0;
  const Tensor scratch = empty({bytes}, at::kByte, logits);
  check(mb200_beam_select(ptr(rows_), fptr(s), static_cast<const uint8_t*>(ptr(f)), ptr(scratch), fptr(out), static_cast<int64_t*>(ptr(tokens)),
                          static_cast<int64_t*>(ptr(parents)), G, B, V, int(std::min<int64_t>(num, 1 << 30)), end_token.value_or(0), stride,
                          dtype_code(dt), cuda_stream()),
        "mb200_beam_select");
  return {out, tokens, parents};
}

Tensor beam_reorder(const Tensor& slots, const Tensor& parents, const std::vector<Tensor>& pools) {
  require_cuda(slots, parents);
  const c10::cuda::CUDAGuard guard(slots.device());
  const BelowAutograd guard_ad;
  TORCH_CHECK(slots.dim() == 2 && parents.sizes() == slots.sizes(), "mamba_b200: slots and parents should both be (groups, beams), got ",
              slots.sizes(), " and ", parents.sizes());
  same_device(slots, {&parents});
  std::vector<void*> at;
  std::vector<int64_t> bytes;
  int64_t n_slots = 0;
  for (const Tensor& p : pools) {
    require_cuda(p);
    same_device(slots, {&p});
    TORCH_CHECK_VALUE(p.dim() >= 1 && p.is_contiguous(), "mamba_b200: pools should be contiguous, because they are updated in place");
    TORCH_CHECK(p.size(0) == pools[0].size(0), "mamba_b200: pools of ", pools[0].size(0), " and ", p.size(0), " slots");
    TORCH_CHECK(!p.requires_grad(), "mamba_b200: pools are updated in place and take no part in automatic differentiation");
    n_slots = p.size(0);
    if (p.numel() == 0) continue;
    at.push_back(p.data_ptr());
    bytes.push_back(int64_t(p.nbytes()) / n_slots);
  }
  const Tensor s = as_type(slots, at::kLong, "slots"), q = as_type(parents, at::kLong, "parents");
  const Tensor out = empty(slots.sizes(), at::kLong, slots);
  check(mb200_beam_reorder(static_cast<const int64_t*>(ptr(s)), static_cast<const int64_t*>(ptr(q)), static_cast<int64_t*>(ptr(out)), slots.size(0),
                           slots.size(1), n_slots, at.data(), bytes.data(), int(at.size()), cuda_stream()),
        "mb200_beam_reorder");
  for (const Tensor& p : pools) written(p);
  return out;
}

}  // namespace mb200_host
