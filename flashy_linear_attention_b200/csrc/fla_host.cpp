// Host side of one forward / backward call on torch tensors: checks, output and scratch tensors,
// argument block and the C-ABI call, in one native function each. Python's part of a call is then a
// few attribute reads; doing the same through torch's Python API and ctypes (about 45 stride reads,
// 40 structure fields and four device guards) took longer than the kernels of a small layer: a
// training step of 8 heads x 256 x 64 took 195 us that way, 95 us this way (18 us of kernels).
//
// Both functions return None for calls they do not cover (wrong types, shapes that do not match,
// head dims above 384, running states with head dims above 128): the caller then takes the general path in
// ops.py, which reports the errors and handles the rest. The interpreter lock is given up while they
// work, as ctypes does: an allocation or a full launch queue can block, and other Python threads, that
// drive other streams or GPUs, have to go on meanwhile.
#include <torch/extension.h>

#include <torch/csrc/autograd/functions/basic_ops.h>

#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <algorithm>
#include <array>
#include <memory>
#include <optional>
#include <string>
#include <vector>

#include "../../include/flashlinear_sm100.h"

namespace {

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

constexpr int64_t kKernelHeadDim = 128;  // widest head dim of the running-state kernels
constexpr int64_t kWideHeadDim = 384;    // widest head dim one library call covers

// What a TMA tensor map needs: unit innermost stride, 16-byte aligned base and outer strides. The row
// stride counts even where there is one row: the library checks it without looking at the length.
bool addressable(const Tensor& t) {
  if (t.stride(3) != 1 || reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 != 0 ||
      t.stride(2) < (t.size(3) + 7) / 8 * 8 || t.stride(2) % 8 != 0)
    return false;
  for (int d = 0; d < 2; ++d)
    if (t.size(d) > 1 && t.stride(d) % 8 != 0) return false;
  return true;
}

bool usable(const Tensor& t, const Tensor& ref) {
  return t.layout() == at::kStrided && t.dim() == 4 && t.is_cuda() && t.device() == ref.device() &&
         t.scalar_type() == ref.scalar_type() && !t.is_neg();
}

bool same_rows(const Tensor& a, const Tensor& b) {  // batch, heads, tokens
  return a.size(0) == b.size(0) && a.size(1) == b.size(1) && a.size(2) == b.size(2);
}

bool is_state(const OptTensor& s, const Tensor& ref, int64_t bh, int64_t dk, int64_t dv) {
  return !s.has_value() || (s->is_cuda() && s->device() == ref.device() && s->scalar_type() == at::kFloat &&
                            s->is_contiguous() && s->dim() == 3 && s->size(0) == bh && s->size(1) == dk &&
                            s->size(2) == dv);
}

FlaTensor desc(const Tensor& t) {
  FlaTensor d;
  d.ptr = t.data_ptr();
  d.stride_b = t.stride(0);
  d.stride_h = t.stride(1);
  d.stride_n = t.stride(2);
  return d;
}

// View [..., :d] of a fresh tensor whose rows are padded to a multiple of 8 elements.
Tensor padded_empty(const Tensor& like) {
  const int64_t d = like.size(3);
  return at::empty({like.size(0), like.size(1), like.size(2), (d + 7) / 8 * 8}, like.options()).narrow(3, 0, d);
}

// empty_like() of a tensor of these sizes and strides that is not at hand any more.
Tensor empty_like_of(const Tensor& sizes_of, at::IntArrayRef strides) {
  const at::IntArrayRef sizes = sizes_of.sizes();
  // strides without gaps or overlaps are kept as they are: walk the dimensions from the inside out
  int order[4] = {3, 2, 1, 0};
  std::stable_sort(order, order + 4, [&](int a, int b) { return strides[a] < strides[b]; });
  int64_t next = 1;
  bool dense = true;
  for (int d : order) {
    if (sizes[d] == 1) continue;
    dense = dense && strides[d] == next;
    next *= sizes[d];
  }
  if (dense) return at::empty_strided(sizes, strides, sizes_of.options());
  return at::empty_like(at::empty_strided(sizes, strides, sizes_of.options().device(at::kMeta)), sizes_of.options());
}

void check(int rc, const char* name) {
  if (rc != FLA_OK)
    throw std::runtime_error(std::string("flashlinear: ") + name + " returned " + std::to_string(rc) + ": " +
                             fla_sm100_strerror(rc));
}

// The library's pad / unpad kernels work on contiguous tensors of any row length.
bool contiguous_rows(const Tensor& t) {
  return t.is_contiguous() && reinterpret_cast<uintptr_t>(t.data_ptr()) % 4 == 0;
}

// Replaces every tensor the kernels cannot address in place by a copy with padded rows. Contiguous
// tensors of one row length share a launch of the pad kernel.
void kernel_views(Tensor* t, int n, void* stream) {
  constexpr int kMax = 4;
  const void* src[kMax];
  void* dst[kMax];
  Tensor copies[kMax];
  bool done[kMax] = {};
  for (int i = 0; i < n; ++i) {
    if (addressable(t[i])) done[i] = true;
    else copies[i] = padded_empty(t[i]);
    if (!done[i] && !contiguous_rows(t[i])) {
      copies[i].copy_(t[i]);
      done[i] = true;
    }
  }
  for (int i = 0; i < n; ++i) {
    if (done[i]) continue;
    int count = 0;
    for (int j = i; j < n; ++j) {
      if (done[j] || t[j].size(3) != t[i].size(3)) continue;
      src[count] = t[j].data_ptr();
      dst[count++] = copies[j].data_ptr();
      done[j] = true;
    }
    check(fla_sm100_pad_rows_batch(src, dst, count, t[i].numel() / t[i].size(3), static_cast<int>(t[i].size(3)),
                                   static_cast<int>(copies[i].stride(2)), stream),
          "fla_sm100_pad_rows_batch");
  }
  for (int i = 0; i < n; ++i)
    if (copies[i].defined()) t[i] = copies[i];
}

// An output with the layout of empty_like(t) and what the kernel writes to: the output itself, or a
// row-padded scratch tensor that is copied back. keep_padded: the padded tensor IS the output.
struct Output {
  Tensor full, view;
};
Output output_like(const Tensor& t, bool keep_padded, const std::vector<int64_t>* strides) {
  Output o;
  if (keep_padded && t.size(3) % 8 != 0) {
    o.full = o.view = padded_empty(t);
    return o;
  }
  o.full = strides != nullptr ? empty_like_of(t, *strides) : at::empty_like(t);
  o.view = addressable(o.full) ? o.full : padded_empty(o.full);
  return o;
}
// Results from the padded scratch rows into the caller-layout outputs, grouped like kernel_views().
void copy_back(const Output* o, int n, void* stream) {
  constexpr int kMax = 4;
  const void* src[kMax];
  void* dst[kMax];
  bool done[kMax] = {};
  for (int i = 0; i < n; ++i) {
    done[i] = o[i].view.is_same(o[i].full);
    if (!done[i] && !contiguous_rows(o[i].full)) {
      o[i].full.copy_(o[i].view);
      done[i] = true;
    }
  }
  for (int i = 0; i < n; ++i) {
    if (done[i]) continue;
    int count = 0;
    const int64_t d = o[i].full.size(3);
    for (int j = i; j < n; ++j) {
      if (done[j] || o[j].full.size(3) != d) continue;
      src[count] = o[j].view.data_ptr();
      dst[count++] = o[j].full.data_ptr();
      done[j] = true;
    }
    check(fla_sm100_unpad_rows_batch(src, dst, count, o[i].full.numel() / d, static_cast<int>(d),
                                     static_cast<int>(o[i].view.stride(2)), stream),
          "fla_sm100_unpad_rows_batch");
  }
}

bool covered_dims(const Tensor& q, const Tensor& v) {
  if (q.numel() == 0 || v.numel() == 0) return false;
  if (q.size(0) > INT32_MAX || q.size(1) > INT32_MAX || q.size(2) > INT32_MAX) return false;
  const int64_t m = std::max(q.size(3), v.size(3));
  if (q.scalar_type() == at::kBFloat16) return m <= kWideHeadDim;
  return q.scalar_type() == at::kHalf && m <= kKernelHeadDim;
}

void set_sizes(FlaArgs& a, const Tensor& q, const Tensor& v, unsigned debug_flags, uintptr_t status) {
  a = FlaArgs{};
  a.batch = static_cast<int32_t>(q.size(0));
  a.heads = static_cast<int32_t>(q.size(1));
  a.seqlen = static_cast<int32_t>(q.size(2));
  a.dk = static_cast<int32_t>(q.size(3));
  a.dv = static_cast<int32_t>(v.size(3));
  a.dtype = q.scalar_type() == at::kHalf ? FLA_DTYPE_F16 : FLA_DTYPE_BF16;
  a.debug_flags = debug_flags;
  a.status = reinterpret_cast<int32_t*>(status);
}

Tensor scratch(FlaArgs& a, int pass, const Tensor& ref) {
  const size_t need = fla_sm100_workspace_bytes(&a, pass);
  if (need == 0) return Tensor();
  Tensor ws = at::empty({static_cast<int64_t>(need)}, ref.options().dtype(at::kByte));
  a.workspace = ws.data_ptr();
  a.workspace_bytes = need;
  return ws;
}

// views: with state 2, the q, k, v the kernels read where
// one of them had to be repacked, for the backward of the same call.
// state: 0 none; 1 always return the final state, [B, H, dk, dv]; 2 return what the backward of
// these shapes uses (final state and boundary states, each a tensor or None).
struct Forward {
  Tensor out;
  OptTensor s_final, seg_states;
  std::optional<std::array<Tensor, 3>> views;
};
std::optional<Forward> forward(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& s_init, int state,
                               unsigned debug_flags, uintptr_t status) {
  if (!usable(q, q) || !usable(k, q) || !usable(v, q) || !covered_dims(q, v) || !same_rows(q, k) ||
      !same_rows(q, v) || q.size(3) != k.size(3))
    return std::nullopt;
  const int64_t bh = q.size(0) * q.size(1), dk = q.size(3), dv = v.size(3);
  const bool wide = dk > kKernelHeadDim || dv > kKernelHeadDim;
  if (wide && (s_init.has_value() || state == 1)) return std::nullopt;
  if (!is_state(s_init, q, bh, dk, dv)) return std::nullopt;
  const c10::cuda::CUDAGuard guard(q.device());
  void* stream = c10::cuda::getCurrentCUDAStream(q.device().index()).stream();
  const Output out = output_like(v, false, nullptr);
  Tensor in[3] = {q, k, v};
  kernel_views(in, 3, stream);
  FlaArgs a;
  set_sizes(a, q, v, debug_flags, status);
  a.stream = stream;
  OptTensor s_final, seg_states;
  if (!wide && (state == 1 || (state == 2 && fla_sm100_bwd_uses_final_state(&a) != 0))) {
    s_final = state == 1 ? at::empty({q.size(0), q.size(1), dk, dv}, q.options().dtype(at::kFloat))
                         : at::empty({bh, dk, dv}, q.options().dtype(at::kFloat));
    if (state == 2) {
      const size_t need = fla_sm100_seg_states_bytes(&a);
      if (need > 0) {
        seg_states = at::empty({static_cast<int64_t>(need)}, q.options().dtype(at::kByte));
        a.seg_states = seg_states->data_ptr();
        a.seg_states_bytes = need;
      }
    }
  }
  a.q = desc(in[0]);
  a.k = desc(in[1]);
  a.v = desc(in[2]);
  a.o = desc(out.view);
  if (s_init.has_value()) a.s_init = s_init->data_ptr<float>();
  if (s_final.has_value()) a.s_final = s_final->data_ptr<float>();
  const Tensor ws = scratch(a, 0, q);
  check(fla_sm100_fwd(&a), "libflashlinear_sm100");
  copy_back(&out, 1, stream);
  Forward res{out.full, s_final, seg_states, std::nullopt};
  if (state == 2 && !(in[0].is_same(q) && in[1].is_same(k) && in[2].is_same(v)))
    res.views = std::array<Tensor, 3>{in[0], in[1], in[2]};
  return res;
}

// strides: those of the three tensors that q, k, v are repacked copies of; the gradients take their layout.
using Strides = std::optional<std::array<std::vector<int64_t>, 3>>;
std::optional<std::array<Tensor, 3>> backward(const Tensor& g, const Tensor& q, const Tensor& k, const Tensor& v,
                                              const OptTensor& s_last, const OptTensor& seg_states, bool keep_padded,
                                              const Strides& strides, unsigned debug_flags, uintptr_t status) {
  Tensor in[4] = {q, k, v, g};
  for (const Tensor& t : in)
    if (!usable(t, q) || !same_rows(t, q)) return std::nullopt;
  if (!covered_dims(q, v) || q.size(3) != k.size(3) || g.size(3) != v.size(3)) return std::nullopt;
  if (strides.has_value())
    for (const auto& s : *strides)
      if (s.size() != 4) return std::nullopt;
  const int64_t bh = q.size(0) * q.size(1), dk = q.size(3), dv = v.size(3);
  if ((dk > kKernelHeadDim || dv > kKernelHeadDim) && s_last.has_value()) return std::nullopt;
  if (!is_state(s_last, g, bh, dk, dv)) return std::nullopt;
  const c10::cuda::CUDAGuard guard(g.device());
  void* stream = c10::cuda::getCurrentCUDAStream(g.device().index()).stream();
  Output out[3];
  for (int i = 0; i < 3; ++i) out[i] = output_like(in[i], keep_padded, strides.has_value() ? &(*strides)[i] : nullptr);
  kernel_views(in, 4, stream);
  FlaArgs a;
  set_sizes(a, q, v, debug_flags, status);
  a.stream = stream;
  a.q = desc(in[0]);
  a.k = desc(in[1]);
  a.v = desc(in[2]);
  a.d_o = desc(in[3]);
  a.d_q = desc(out[0].view);
  a.d_k = desc(out[1].view);
  a.d_v = desc(out[2].view);
  if (s_last.has_value()) a.s_last = s_last->data_ptr<float>();
  if (seg_states.has_value()) {
    a.seg_states = seg_states->data_ptr();
    a.seg_states_bytes = static_cast<size_t>(seg_states->numel() * seg_states->element_size());
  }
  const Tensor ws = scratch(a, 1, g);
  check(fla_sm100_bwd(&a), "libflashlinear_sm100");
  copy_back(out, 3, stream);
  return std::array<Tensor, 3>{out[0].full, out[1].full, out[2].full};
}

// Attention on the Taylor features of raw q, k.
bool taylor_covered(const Tensor& q, const Tensor& k, const Tensor& v) {
  const int64_t d = q.dim() == 4 ? q.size(3) : 0, dv = v.dim() == 4 ? v.size(3) : 0;
  return usable(q, q) && usable(k, q) && usable(v, q) && same_rows(q, k) && same_rows(q, v) && k.size(3) == d &&
         (d == 8 || d == 16) && (dv == 8 || dv == 16 || dv == 32 || dv == 64) && q.scalar_type() == at::kBFloat16 && covered_dims(q, v);
}
std::optional<Tensor> taylor_forward(const Tensor& q, const Tensor& k, const Tensor& v, unsigned debug_flags, uintptr_t status) {
  if (!taylor_covered(q, k, v)) return std::nullopt;
  const c10::cuda::CUDAGuard guard(q.device());
  void* stream = c10::cuda::getCurrentCUDAStream(q.device().index()).stream();
  const Output out = output_like(v, false, nullptr);
  Tensor in[3] = {q, k, v};
  kernel_views(in, 3, stream);
  FlaArgs a;
  set_sizes(a, q, v, debug_flags, status);
  a.stream = stream;
  a.q = desc(in[0]);
  a.k = desc(in[1]);
  a.v = desc(in[2]);
  a.o = desc(out.view);
  check(fla_sm100_taylor_fwd(&a), "fla_sm100_taylor_fwd");
  copy_back(&out, 1, stream);
  return out.full;
}
std::optional<std::array<Tensor, 3>> taylor_backward(const Tensor& g, const Tensor& q, const Tensor& k, const Tensor& v,
                                                     unsigned debug_flags, uintptr_t status) {
  if (!taylor_covered(q, k, v) || !usable(g, q) || !same_rows(g, q) || g.size(3) != v.size(3)) return std::nullopt;
  const c10::cuda::CUDAGuard guard(g.device());
  void* stream = c10::cuda::getCurrentCUDAStream(g.device().index()).stream();
  const Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options());
  const Output dv = output_like(v, false, nullptr);
  Tensor in[4] = {q, k, v, g};
  kernel_views(in, 4, stream);
  FlaArgs a;
  set_sizes(a, q, v, debug_flags, status);
  a.stream = stream;
  a.q = desc(in[0]);
  a.k = desc(in[1]);
  a.v = desc(in[2]);
  a.d_o = desc(in[3]);
  a.d_q = desc(dq);
  a.d_k = desc(dk);
  a.d_v = desc(dv.view);
  check(fla_sm100_taylor_bwd(&a), "fla_sm100_taylor_bwd");
  copy_back(&dv, 1, stream);
  return std::array<Tensor, 3>{dq, dk, dv.full};
}

// The same through features in memory: out and the features of q and k, rows padded to a multiple of 8
// elements; and the gradients from those. (Prepared in Python a training step took 200 us of the host.)
struct FeatureDims {
  int features, padded;
};
std::optional<FeatureDims> feature_dims(const Tensor& q, const Tensor& k, const Tensor& v) {
  FeatureDims f;
  if (!usable(q, q) || !usable(k, q) || !usable(v, q) || q.sizes() != k.sizes() || !same_rows(q, v) ||
      q.scalar_type() != at::kBFloat16 || !covered_dims(q, v) ||
      fla_sm100_taylor_dims(static_cast<int>(q.size(3)), &f.features, &f.padded) != FLA_OK)
    return std::nullopt;
  return f;
}
Tensor aligned_rows(const Tensor& x) {  // what the feature kernels read
  const Tensor c = x.contiguous();
  return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 == 0 ? c : c.clone();
}
std::optional<std::array<Tensor, 3>> taylor_forward_in_memory(const Tensor& q, const Tensor& k, const Tensor& v,
                                                              unsigned debug_flags, uintptr_t status) {
  const auto dims = feature_dims(q, k, v);
  if (!dims.has_value()) return std::nullopt;
  const c10::cuda::CUDAGuard guard(q.device());
  void* stream = c10::cuda::getCurrentCUDAStream(q.device().index()).stream();
  auto features = [&](const Tensor& x) {
    const Tensor rows = aligned_rows(x);
    const Tensor phi = at::empty({x.size(0), x.size(1), x.size(2), dims->padded}, x.options());
    check(fla_sm100_taylor_features(rows.data_ptr(), phi.data_ptr(), x.numel() / x.size(3), static_cast<int>(x.size(3)), stream),
          "fla_sm100_taylor_features");
    return phi.narrow(3, 0, dims->features);
  };
  const Tensor pq = features(q), pk = features(k);
  const std::optional<Forward> r = forward(pq, pk, v, std::nullopt, 0, debug_flags, status);
  if (!r.has_value()) return std::nullopt;
  return std::array<Tensor, 3>{r->out, pq, pk};
}
std::optional<std::array<Tensor, 3>> taylor_backward_in_memory(const Tensor& g, const Tensor& q, const Tensor& k,
                                                               const Tensor& v, const Tensor& pq, const Tensor& pk,
                                                               unsigned debug_flags, uintptr_t status) {
  const auto dims = feature_dims(q, k, v);
  if (!dims.has_value()) return std::nullopt;
  const auto r = backward(g, pq, pk, v, std::nullopt, std::nullopt, true, std::nullopt, debug_flags, status);
  if (!r.has_value()) return std::nullopt;
  const c10::cuda::CUDAGuard guard(q.device());
  void* stream = c10::cuda::getCurrentCUDAStream(q.device().index()).stream();
  auto raw = [&](const Tensor& dphi, const Tensor& x) {  // (dphi: fresh, its rows padded as those of the features)
    const Tensor rows = aligned_rows(x), dx = at::empty(x.sizes(), x.options());
    check(fla_sm100_taylor_features_bwd(dphi.data_ptr(), rows.data_ptr(), dx.data_ptr(), x.numel() / x.size(3),
                                        static_cast<int>(x.size(3)), stream),
          "fla_sm100_taylor_features_bwd");
    return dx;
  };
  return std::array<Tensor, 3>{raw((*r)[0], q), raw((*r)[1], k), (*r)[2]};
}

// The gated linear recurrence. Tensors are read where they are; neighbouring columns have to be neighbours in memory.
bool recurrence_rows(const Tensor& t) {
  return t.layout() == at::kStrided && t.dim() == 4 && t.is_cuda() && !t.is_neg() && (t.stride(3) == 1 || t.size(3) == 1);
}
int float_type(const Tensor& t) {
  const auto s = t.scalar_type();
  return s == at::kBFloat16 ? FLA_DTYPE_BF16 : s == at::kHalf ? FLA_DTYPE_F16 : s == at::kFloat ? FLA_DTYPE_F32 : -1;
}
bool recurrence_covered(const Tensor& x, const Tensor& g) {
  if (!recurrence_rows(x) || !recurrence_rows(g) || x.sizes() != g.sizes() || x.device() != g.device() || x.numel() == 0)
    return false;
  if (float_type(x) < 0 || (float_type(g) != float_type(x) && float_type(g) != FLA_DTYPE_F32)) return false;
  constexpr int64_t kMost = 1 << 30;
  return x.size(0) <= kMost && x.size(1) <= kMost && x.size(0) * x.size(1) <= kMost && x.size(2) <= kMost && x.size(3) <= kMost;
}
bool channel_state(const OptTensor& s, const Tensor& x) {
  return !s.has_value() || (s->is_cuda() && s->device() == x.device() && s->scalar_type() == at::kFloat && s->dim() == 3 &&
                            s->size(0) == x.size(0) && s->size(1) == x.size(1) && s->size(2) == x.size(3) &&
                            s->is_contiguous() && !s->is_neg());
}
Tensor rows_like(const Tensor& t) {
  const Tensor out = at::empty_like(t);
  return recurrence_rows(out) ? out : at::empty(t.sizes(), t.options());
}
FlaRecurrenceArgs recurrence_args(const Tensor& x, const Tensor& g, unsigned debug_flags, uintptr_t status) {
  FlaRecurrenceArgs a = {};
  a.batch = static_cast<int32_t>(x.size(0));
  a.heads = static_cast<int32_t>(x.size(1));
  a.seqlen = static_cast<int32_t>(x.size(2));
  a.dim = static_cast<int32_t>(x.size(3));
  a.dtype = float_type(x);
  a.g_dtype = float_type(g);
  a.x = desc(x);
  a.g = desc(g);
  a.debug_flags = debug_flags;
  a.status = reinterpret_cast<int32_t*>(status);
  a.stream = c10::cuda::getCurrentCUDAStream(x.device().index()).stream();
  return a;
}
struct Recurrence {
  Tensor out, s_final;
  OptTensor states;
};
std::optional<Recurrence> recurrence_forward(const Tensor& x, const Tensor& g, const OptTensor& s_init, bool keep_states,
                                             unsigned debug_flags, uintptr_t status) {
  if (!recurrence_covered(x, g) || !channel_state(s_init, x)) return std::nullopt;
  const c10::cuda::CUDAGuard guard(x.device());
  FlaRecurrenceArgs a = recurrence_args(x, g, debug_flags, status);
  Recurrence r{rows_like(x), at::empty({x.size(0), x.size(1), x.size(3)}, x.options().dtype(at::kFloat)), std::nullopt};
  a.o = desc(r.out);
  if (s_init.has_value()) a.s_init = s_init->data_ptr<float>();
  a.s_final = r.s_final.data_ptr<float>();
  if (keep_states) {
    a.states_bytes = fla_sm100_recurrence_states_bytes(&a);
    r.states = at::empty({static_cast<int64_t>(a.states_bytes)}, x.options().dtype(at::kByte));
    a.states = r.states->data_ptr();
  }
  check(fla_sm100_recurrence_fwd(&a), "fla_sm100_recurrence_fwd");
  return r;
}
std::optional<std::array<OptTensor, 3>> recurrence_backward(const OptTensor& dy, const Tensor& x, const Tensor& g,
                                                            const OptTensor& states, const OptTensor& ds, bool need_x,
                                                            bool need_g, bool need_s, unsigned debug_flags, uintptr_t status) {
  if (!recurrence_covered(x, g) || !channel_state(ds, x) || !states.has_value() || !states->is_cuda() ||
      states->device() != x.device() || !states->is_contiguous() || !(need_x || need_g || need_s))
    return std::nullopt;
  const c10::cuda::CUDAGuard guard(x.device());
  FlaRecurrenceArgs a = recurrence_args(x, g, debug_flags, status);
  Tensor rows;
  if (dy.has_value()) {
    if (dy->sizes() != x.sizes() || dy->scalar_type() != x.scalar_type() || dy->device() != x.device()) return std::nullopt;
    rows = recurrence_rows(*dy) ? *dy : dy->resolve_neg().contiguous();
    if (!recurrence_rows(rows)) return std::nullopt;
    a.d_o = desc(rows);
  }
  std::array<OptTensor, 3> out;
  if (need_x) a.d_x = desc(*(out[0] = rows_like(x)));
  if (need_g) a.d_g = desc(*(out[1] = rows_like(g)));
  if (need_s) a.r_final = (out[2] = at::empty({x.size(0), x.size(1), x.size(3)}, x.options().dtype(at::kFloat)))->data_ptr<float>();
  if (ds.has_value()) a.r_init = ds->data_ptr<float>();
  a.states = states->data_ptr();
  a.states_bytes = static_cast<size_t>(states->numel() * states->element_size());
  check(fla_sm100_recurrence_bwd(&a), "fla_sm100_recurrence_bwd");
  return out;
}

// Layer norm, of rows in up to four dimensions.
bool norm_rows(const Tensor& t, const Tensor& x) {
  return t.layout() == at::kStrided && t.dim() >= 1 && t.dim() <= 4 && t.is_cuda() && t.device() == x.device() && !t.is_neg() &&
         t.sizes() == x.sizes() && t.scalar_type() == x.scalar_type() && (t.stride(-1) == 1 || t.size(-1) == 1);
}
bool norm_weights(const OptTensor& w, const Tensor& x) {
  if (!w.has_value()) return true;
  if (!w->is_cuda() || w->device() != x.device() || !w->is_contiguous() || w->is_neg()) return false;
  if (w->dim() < 1 || w->size(-1) != x.size(-1)) return false;
  if (w->dim() != 1 && !(w->dim() == 2 && x.dim() == 4 && w->size(0) == x.size(1))) return false;
  return float_type(*w) == float_type(x) || float_type(*w) == FLA_DTYPE_F32;
}
bool norm_covered(const Tensor& x, const OptTensor& w, const OptTensor& b) {
  if (!norm_rows(x, x) || float_type(x) < 0 || x.numel() == 0 || x.size(-1) > 32768 || x.numel() / x.size(-1) > INT32_MAX)
    return false;
  if (!norm_weights(w, x) || !norm_weights(b, x)) return false;
  return !w.has_value() || !b.has_value() || (w->sizes() == b->sizes() && w->scalar_type() == b->scalar_type());
}
FlaTensor norm_desc(const Tensor& t) {  // [B, H, N, D], [B, N, D], [N, D] or [D]
  const int64_t n = t.dim();
  FlaTensor d = {};
  d.ptr = t.data_ptr();
  if (n >= 2) d.stride_n = t.stride(n - 2);
  if (n == 4) d.stride_h = t.stride(1);
  if (n >= 3) d.stride_b = t.stride(0);
  return d;
}
Tensor norm_like(const Tensor& t) {
  const Tensor out = at::empty_like(t);
  return norm_rows(out, t) ? out : at::empty(t.sizes(), t.options());
}
FlaLayerNormArgs norm_args(const Tensor& x, const OptTensor& w, const OptTensor& b, double eps) {
  const int64_t n = x.dim();
  FlaLayerNormArgs a = {};
  a.batch = n >= 3 ? static_cast<int32_t>(x.size(0)) : 1;
  a.heads = n == 4 ? static_cast<int32_t>(x.size(1)) : 1;
  a.tokens = n >= 2 ? static_cast<int32_t>(x.size(n - 2)) : 1;
  a.dim = static_cast<int32_t>(x.size(n - 1));
  a.dtype = a.w_dtype = float_type(x);
  for (const OptTensor* t : {&w, &b})
    if (t->has_value()) {
      a.w_dtype = float_type(**t);
      a.per_head = (*t)->dim() == 2;
    }
  a.eps = static_cast<float>(eps);
  a.x = norm_desc(x);
  if (w.has_value()) a.weight = w->data_ptr();
  if (b.has_value()) a.bias = b->data_ptr();
  a.stream = c10::cuda::getCurrentCUDAStream(x.device().index()).stream();
  return a;
}
struct Norm {
  Tensor out;
  OptTensor sum, stats;
};
std::optional<Norm> layer_norm_forward(const Tensor& x, const OptTensor& w, const OptTensor& b, double eps,
                                       const OptTensor& residual, bool keep_stats) {
  if (!norm_covered(x, w, b) || (residual.has_value() && !norm_rows(*residual, x)) || !(eps >= 0)) return std::nullopt;
  const c10::cuda::CUDAGuard guard(x.device());
  FlaLayerNormArgs a = norm_args(x, w, b, eps);
  Norm r{norm_like(x), std::nullopt, std::nullopt};
  a.y = norm_desc(r.out);
  if (residual.has_value()) {
    r.sum = norm_like(x);
    a.residual = norm_desc(*residual);
    a.sum = norm_desc(*r.sum);
  }
  if (keep_stats) {
    r.stats = at::empty({x.numel() / x.size(-1), 2}, x.options().dtype(at::kFloat));
    a.stats = r.stats->data_ptr<float>();
  }
  check(fla_sm100_layer_norm_fwd(&a), "fla_sm100_layer_norm_fwd");
  return r;
}
std::optional<std::array<OptTensor, 3>> layer_norm_backward(const Tensor& dy, const Tensor& x, const OptTensor& w, const OptTensor& b,
                                                            const Tensor& stats, const OptTensor& ds, bool need_x, bool need_w,
                                                            bool need_b) {
  if (!norm_covered(x, w, b) || !norm_rows(dy, x) || (ds.has_value() && !norm_rows(*ds, x)) || !stats.is_cuda() ||
      stats.device() != x.device() || stats.scalar_type() != at::kFloat || !stats.is_contiguous() ||
      stats.numel() != 2 * (x.numel() / x.size(-1)) || !(need_x || need_w || need_b))
    return std::nullopt;
  const c10::cuda::CUDAGuard guard(x.device());
  FlaLayerNormArgs a = norm_args(x, w, b, 0.0);
  a.d_y = norm_desc(dy);
  if (ds.has_value()) a.d_sum = norm_desc(*ds);
  a.stats = stats.data_ptr<float>();
  std::array<OptTensor, 3> out;
  if (need_x) a.d_x = norm_desc(*(out[0] = norm_like(x)));
  if (need_w) a.d_weight = (out[1] = at::empty(w->sizes(), w->options()))->data_ptr();
  if (need_b) a.d_bias = (out[2] = at::empty(b->sizes(), b->options()))->data_ptr();
  Tensor ws;
  if (const size_t need = fla_sm100_layer_norm_workspace_bytes(&a)) {
    ws = at::empty({static_cast<int64_t>(need)}, x.options().dtype(at::kByte));
    a.workspace = ws.data_ptr();
    a.workspace_bytes = need;
  }
  check(fla_sm100_layer_norm_bwd(&a), "fla_sm100_layer_norm_bwd");
  return out;
}

// The Functions around these calls as native autograd nodes: a backward in Python has to be handed the interpreter lock by the
// thread that waits for it, and a training step of a small layer took 90 us that way, of which 20 are these calls. The first
// value of a result is empty where the call is not covered: the caller then takes the Python Functions of the same names.
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Gradients are not differentiable themselves; the error comes when somebody tries.
variable_list once_differentiable(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  for (Tensor& g : grads) {
    if (!g.defined()) continue;
    const auto error = std::make_shared<torch::autograd::DelayedError>(
        "trying to differentiate twice a function that was marked with @once_differentiable", 1);
    Tensor leaf = g.detach();
    leaf.set_requires_grad(true);
    g = error->apply({leaf})[0];
  }
  return grads;
}
bool wants_gradient(const Tensor& x, std::initializer_list<const OptTensor*> others) {
  if (!at::GradMode::is_enabled()) return false;
  for (const OptTensor* t : others)
    if (t->has_value() && (*t)->requires_grad()) return true;
  return x.requires_grad();
}
Tensor or_none(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
OptTensor or_null(const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; }

struct RecurrenceNode : torch::autograd::Function<RecurrenceNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& g, const OptTensor& s_init, bool keep,
                               int64_t debug_flags, int64_t status) {
    const auto r = recurrence_forward(x, g, s_init, keep, static_cast<unsigned>(debug_flags), static_cast<uintptr_t>(status));
    if (!r.has_value()) throw std::runtime_error("flashlinear: the recurrence's arguments changed between two checks");
    if (keep) {
      ctx->save_for_backward({x, g, or_none(r->states)});
      ctx->saved_data["flags"] = debug_flags;
      ctx->saved_data["status"] = status;
      ctx->saved_data["wants"] = static_cast<int64_t>(x.requires_grad()) | static_cast<int64_t>(g.requires_grad()) << 1 |
                                 static_cast<int64_t>(s_init.has_value() && s_init->requires_grad()) << 2;
    }
    ctx->set_materialize_grads(false);
    return {r->out, r->s_final};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    variable_list out(6);
    if (!grads[0].defined() && !grads[1].defined()) return out;
    const variable_list saved = ctx->get_saved_variables();
    const int64_t wants = ctx->saved_data["wants"].toInt();
    {
      const at::AutoGradMode off(false);
      const Tensor ds = grads[1].defined() ? grads[1].resolve_neg().to(at::kFloat).contiguous() : Tensor();
      const auto r = recurrence_backward(or_null(grads[0]), saved[0], saved[1], saved[2], or_null(ds), wants & 1, wants & 2, wants & 4,
                                         static_cast<unsigned>(ctx->saved_data["flags"].toInt()),
                                         static_cast<uintptr_t>(ctx->saved_data["status"].toInt()));
      if (!r.has_value()) throw std::runtime_error("flashlinear: the gradients of the recurrence's outputs do not fit them");
      for (int i = 0; i < 3; ++i) out[i] = or_none((*r)[i]);
    }
    return once_differentiable(std::move(out));
  }
};

// LayerNorm without, AddLayerNorm with a residual.
struct LayerNormNode : torch::autograd::Function<LayerNormNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptTensor& residual, const OptTensor& w, const OptTensor& b,
                               double eps, bool keep) {
    const auto r = layer_norm_forward(x, w, b, eps, residual, keep);
    if (!r.has_value()) throw std::runtime_error("flashlinear: the layer norm's arguments changed between two checks");
    if (keep) {
      ctx->save_for_backward({residual.has_value() ? *r->sum : x, or_none(w), or_none(b), or_none(r->stats)});
      ctx->saved_data["wants"] = static_cast<int64_t>(x.requires_grad() || (residual.has_value() && residual->requires_grad())) |
                                 static_cast<int64_t>(w.has_value() && w->requires_grad()) << 1 |
                                 static_cast<int64_t>(b.has_value() && b->requires_grad()) << 2;
      ctx->saved_data["residual"] = residual.has_value();
    }
    ctx->set_materialize_grads(false);
    if (residual.has_value()) return {r->out, *r->sum};
    return {r->out};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    variable_list out(6);
    const bool residual = ctx->saved_data["residual"].toBool();
    const Tensor ds = residual ? grads[1] : Tensor();
    if (!grads[0].defined()) {  // the sum alone was used
      out[0] = out[1] = ds;
      return out;
    }
    const variable_list saved = ctx->get_saved_variables();
    const int64_t wants = ctx->saved_data["wants"].toInt();
    {
      const at::AutoGradMode off(false);
      auto rows = [&](const Tensor& t) { return !t.defined() || norm_rows(t, saved[0]) ? t : t.resolve_neg().contiguous(); };
      const auto r = layer_norm_backward(rows(grads[0]), saved[0], or_null(saved[1]), or_null(saved[2]), saved[3], or_null(rows(ds)),
                                         wants & 1, wants & 2, wants & 4);
      if (!r.has_value()) throw std::runtime_error("flashlinear: the gradients of the layer norm's outputs do not fit them");
      out[0] = or_none((*r)[0]);
      if (residual) out[1] = out[0];
      out[2] = or_none((*r)[1]);
      out[3] = or_none((*r)[2]);
    }
    return once_differentiable(std::move(out));
  }
};

variable_list recurrence_apply(const Tensor& x, const Tensor& g, const OptTensor& s_init, unsigned debug_flags, uintptr_t status) {
  if (!recurrence_covered(x, g) || !channel_state(s_init, x)) return {};
  return RecurrenceNode::apply(x, g, s_init, g.requires_grad() && at::GradMode::is_enabled() ? true : wants_gradient(x, {&s_init}),
                               static_cast<int64_t>(debug_flags), static_cast<int64_t>(status));
}
variable_list layer_norm_apply(const Tensor& x, const OptTensor& residual, const OptTensor& w, const OptTensor& b, double eps) {
  if (!norm_covered(x, w, b) || (residual.has_value() && !norm_rows(*residual, x)) || !(eps >= 0)) return {};
  return LayerNormNode::apply(x, residual, w, b, eps, wants_gradient(x, {&residual, &w, &b}));
}

// What is saved beside the repacked copy of an input that is not kept itself: an empty tensor that shares
// its version count, for autograd to see that it was changed in place. (An inference tensor has none;
// it is returned itself, and autograd refuses it as it always does.)
Tensor version_of(const Tensor& t) {
  if (t.is_inference()) return t;
  const Tensor version = at::empty({0}, t.options());
  torch::autograd::impl::set_version_counter(version, torch::autograd::impl::version_counter(t));
  return version;
}

}  // namespace

PYBIND11_MODULE(_hostcalls, m) {
  m.attr("abi_version") = FLA_ABI_VERSION;
  m.def("forward", [](const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& s_init, int state,
                      unsigned debug_flags, uintptr_t status) -> py::object {
    std::optional<Forward> r;
    {
      const py::gil_scoped_release unlocked;
      r = forward(q, k, v, s_init, state, debug_flags, status);
    }
    if (!r.has_value()) return py::none();
    py::object views = py::none();
    if (r->views.has_value()) views = py::make_tuple((*r->views)[0], (*r->views)[1], (*r->views)[2]);
    return py::make_tuple(r->out, r->s_final, r->seg_states, views);
  });
  m.def("version_of", &version_of);
  m.def("recurrence_apply", &recurrence_apply, py::call_guard<py::gil_scoped_release>());
  m.def("layer_norm_apply", &layer_norm_apply, py::call_guard<py::gil_scoped_release>());
  m.def("layer_norm_forward", [](const Tensor& x, const OptTensor& w, const OptTensor& b, double eps, const OptTensor& residual,
                                 bool keep_stats) -> py::object {
    std::optional<Norm> r;
    {
      const py::gil_scoped_release unlocked;
      r = layer_norm_forward(x, w, b, eps, residual, keep_stats);
    }
    if (!r.has_value()) return py::none();
    return py::make_tuple(r->out, r->sum, r->stats);
  });
  m.def("layer_norm_backward", [](const Tensor& dy, const Tensor& x, const OptTensor& w, const OptTensor& b, const Tensor& stats,
                                  const OptTensor& ds, bool need_x, bool need_w, bool need_b) -> py::object {
    std::optional<std::array<OptTensor, 3>> r;
    {
      const py::gil_scoped_release unlocked;
      r = layer_norm_backward(dy, x, w, b, stats, ds, need_x, need_w, need_b);
    }
    if (!r.has_value()) return py::none();
    return py::make_tuple((*r)[0], (*r)[1], (*r)[2]);
  });
  m.def("recurrence_forward", [](const Tensor& x, const Tensor& g, const OptTensor& s_init, bool keep_states,
                                 unsigned debug_flags, uintptr_t status) -> py::object {
    std::optional<Recurrence> r;
    {
      const py::gil_scoped_release unlocked;
      r = recurrence_forward(x, g, s_init, keep_states, debug_flags, status);
    }
    if (!r.has_value()) return py::none();
    return py::make_tuple(r->out, r->s_final, r->states);
  });
  m.def("recurrence_backward", [](const OptTensor& dy, const Tensor& x, const Tensor& g, const OptTensor& states,
                                  const OptTensor& ds, bool need_x, bool need_g, bool need_s, unsigned debug_flags,
                                  uintptr_t status) -> py::object {
    std::optional<std::array<OptTensor, 3>> r;
    {
      const py::gil_scoped_release unlocked;
      r = recurrence_backward(dy, x, g, states, ds, need_x, need_g, need_s, debug_flags, status);
    }
    if (!r.has_value()) return py::none();
    return py::make_tuple((*r)[0], (*r)[1], (*r)[2]);
  });
  m.def("taylor_forward", &taylor_forward, py::call_guard<py::gil_scoped_release>());
  m.def("taylor_backward", &taylor_backward, py::call_guard<py::gil_scoped_release>());
  m.def("taylor_forward_in_memory", &taylor_forward_in_memory, py::call_guard<py::gil_scoped_release>());
  m.def("taylor_backward_in_memory", &taylor_backward_in_memory, py::call_guard<py::gil_scoped_release>());
  m.def("backward", [](const Tensor& g, const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& s_last,
                       const OptTensor& seg_states, bool keep_padded, const Strides& strides, unsigned debug_flags,
                       uintptr_t status) -> py::object {
    std::optional<std::array<Tensor, 3>> r;
    {
      const py::gil_scoped_release unlocked;
      r = backward(g, q, k, v, s_last, seg_states, keep_padded, strides, debug_flags, status);
    }
    if (!r.has_value()) return py::none();
    return py::make_tuple((*r)[0], (*r)[1], (*r)[2]);
  });
}
