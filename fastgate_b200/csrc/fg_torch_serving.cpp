// pybind11 / torch-extension surface of the operators that stand around the linears in a serving step: RMS norm,
// linear on 8-bit activations, 4-bit key/value cache.  Thin layers over the C ABI, like fg_torch.cpp: tensor checks, the current
// stream of the tensors' device, workspaces, status codes as exceptions.  There is no CPU path.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_runtime.h>
#include <torch/extension.h>

#include <map>
#include <mutex>
#include <stdexcept>
#include <string>
#include <utility>

#include "../../include/fastgate_b200.h"
#include "fg_torch.h"

namespace {

using OptTensor = c10::optional<at::Tensor>;

bool given(const OptTensor& t) { return t.has_value() && t->defined(); }

[[noreturn]] void bad_argument(const std::string& what) { throw std::invalid_argument("fastgate_b200: " + what); }

void check_status(int st) {
  if (st == FG_OK) return;
  const std::string text = std::string("fastgate_b200: ") + fg_status_str(st);
  if (st == FG_ERR_SHAPE) throw std::invalid_argument("fastgate_b200: sizes or strides are out of the operator's range");
  if (st == FG_ERR_ALIGN) throw std::invalid_argument(text);
  throw std::runtime_error(text + " (cuda error " + std::to_string(fg_last_cuda_error()) + ")");
}

// A CUDA tensor of type `dt` on `device` (-1: any).
void check_cuda(const at::Tensor& t, const char* name, at::ScalarType dt, int64_t device) {
  if (!t.defined()) bad_argument(std::string(name) + " is missing");
  if (!t.is_cuda()) throw std::runtime_error(std::string("fastgate_b200: ") + name + " must be a CUDA tensor (there is no CPU path)");
  if (t.scalar_type() != dt) throw std::runtime_error(std::string("fastgate_b200: ") + name + " has the wrong dtype");
  if (device >= 0 && t.get_device() != device) throw std::runtime_error("fastgate_b200: all tensors must live on one device");
}
void check_dense(const at::Tensor& t, const char* name, at::ScalarType dt, int64_t device) {
  check_cuda(t, name, dt, device);
  if (!t.is_contiguous()) throw std::runtime_error(std::string("fastgate_b200: ") + name + " must be contiguous");
}
// [rows, heads, d] with dense heads and any row stride.
void check_rows(const at::Tensor& t, const char* name, int64_t device) {
  check_cuda(t, name, at::kHalf, device);
  if (t.dim() != 3) bad_argument(std::string(name) + " must be [tokens, heads, channels]");
  if ((t.size(2) > 1 && t.stride(2) != 1) || (t.size(1) > 1 && t.stride(1) != t.size(2)))
    bad_argument(std::string(name) + " must have dense heads and channels (only the token stride is free)");
}
// Distance between rows; a single row's is whatever makes the check on it pass.
int64_t row_stride(const at::Tensor& t) {
  const int64_t dense = t.dim() == 3 ? t.size(1) * t.size(2) : t.size(1);
  return t.size(0) > 1 ? t.stride(0) : dense;
}
// A one-dimensional int32 or int64 index tensor of n elements; returns whether it is int64.
int check_index(const at::Tensor& t, const char* name, int64_t n, int64_t device) {
  if (t.defined() && t.is_cuda() && t.scalar_type() == at::kInt) check_dense(t, name, at::kInt, device);
  else check_dense(t, name, at::kLong, device);
  if (t.dim() != 1 || t.size(0) != n) bad_argument(std::string(name) + " must hold one index per token");
  return t.scalar_type() == at::kLong;
}
int* status_ptr(const OptTensor& status, int64_t device) {
  if (!given(status)) return nullptr;
  check_dense(*status, "status", at::kInt, device);
  if (status->numel() < 1) bad_argument("status must hold one int32");
  return status->data_ptr<int>();
}
bool overlap(const at::Tensor& a, const at::Tensor& b) {
  auto end = [](const at::Tensor& t) {
    int64_t last = 0;
    for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
    return static_cast<const char*>(t.data_ptr()) + (last + 1) * t.element_size();
  };
  if (a.numel() == 0 || b.numel() == 0) return false;
  return static_cast<const char*>(a.data_ptr()) < end(b) && static_cast<const char*>(b.data_ptr()) < end(a);
}

// The same for tensors of rows that are dense in themselves ([tokens, heads, channels], or anything dense): column ranges of one
// buffer lie between each other's rows without meeting them.
bool rows_overlap(const at::Tensor& a, const at::Tensor& b) {
  if (!overlap(a, b)) return false;
  if (a.dim() != 3 || b.dim() != 3 || a.size(0) < 2 || b.size(0) < 2 || a.element_size() != b.element_size() || a.stride(0) != b.stride(0)) return true;
  const int64_t size = a.element_size(), step = a.stride(0) * size;
  const int64_t wa = a.size(1) * a.size(2) * size, wb = b.size(1) * b.size(2) * size;
  if (step < wa || step < wb) return true;
  // where b's rows begin within a's period
  const int64_t d = static_cast<const char*>(b.data_ptr()) - static_cast<const char*>(a.data_ptr());
  const int64_t at = (d % step + step) % step;
  return at < wa || at + wb > step;
}

// ---- RMS norm ------------------------------------------------------------------------------
void add_rmsnorm(at::Tensor x, at::Tensor weight, at::Tensor out, OptTensor residual, double eps, OptTensor scales, OptTensor residual_out) {
  check_cuda(x, "x", at::kHalf, -1);
  const int64_t device = x.get_device();
  if (x.dim() != 2 || (x.size(1) > 1 && x.stride(1) != 1)) bad_argument("x must be [M, K] with dense rows");
  const int64_t M = x.size(0), K = x.size(1);
  check_dense(weight, "weight", at::kHalf, device);
  if (weight.dim() != 1 || weight.size(0) != K) bad_argument("weight must hold K elements");
  const bool int8 = out.defined() && out.scalar_type() == at::kChar;
  check_dense(out, "out", int8 ? at::kChar : at::kHalf, device);
  if (out.dim() != 2 || out.sizes() != x.sizes()) bad_argument("out must have the shape of x");
  if (int8 != given(scales)) bad_argument(int8 ? "an int8 out needs scales" : "scales go with an int8 out");
  if (int8) {
    check_dense(*scales, "scales", at::kFloat, device);
    if (scales->numel() != M) bad_argument("scales must hold one fp32 value per row");
    if (overlap(*scales, x) || overlap(*scales, out) || overlap(*scales, weight) || (given(residual) && overlap(*scales, *residual)) ||
        (given(residual_out) && overlap(*scales, *residual_out)))
      bad_argument("scales must not overlap the other buffers");
  }
  const void* res = nullptr;
  void* res_out = nullptr;
  int f32 = 0;
  if (given(residual)) {
    f32 = residual->scalar_type() == at::kFloat;
    const at::ScalarType dt = f32 ? at::kFloat : at::kHalf;
    check_dense(*residual, "residual", dt, device);
    if (residual->sizes() != x.sizes()) bad_argument("residual must have the shape of x");
    at::Tensor ro = given(residual_out) ? *residual_out : *residual;
    check_dense(ro, "residual_out", dt, device);
    if (ro.sizes() != x.sizes()) bad_argument("residual_out must have the shape of x");
    res = residual->data_ptr();
    res_out = ro.data_ptr();
    if ((ro.data_ptr() != residual->data_ptr() && overlap(ro, *residual)) || overlap(ro, x) || overlap(ro, out) || overlap(ro, weight) ||
        overlap(*residual, out))
      bad_argument("residual_out may be residual itself; otherwise the buffers must not overlap");
  } else if (given(residual_out)) {
    bad_argument("residual_out without residual");
  }
  if (overlap(out, weight) || (overlap(out, x) && !(!int8 && x.is_contiguous() && out.data_ptr() == x.data_ptr())))
    bad_argument("an fp16 out may be x itself; otherwise the buffers must not overlap");
  if (!(eps >= 0) || K == 0 || (K % 8) != 0) bad_argument("K must be a multiple of 8 and eps not negative");
  if (M == 0) return;
  if (M > 0x7fffffff || K > 0x7fffffff) bad_argument("x is too large");
  if (row_stride(x) % 8 != 0) bad_argument("the row stride of x must be a multiple of 8 elements");
  const c10::cuda::CUDAGuard guard(x.device());
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(device).stream();
  int st;
  {
    pybind11::gil_scoped_release nogil;
    st = fg_add_rmsnorm(x.data_ptr(), row_stride(x), weight.data_ptr(), res, res_out, f32, out.data_ptr(), int8,
                        int8 ? scales->data_ptr<float>() : nullptr, static_cast<int>(M), static_cast<int>(K), static_cast<float>(eps),
                        reinterpret_cast<fg_stream_t>(stream));
  }
  check_status(st);
}

// ---- linear on 8-bit activations -------------------------------------------------------------
void linear_int8(at::Tensor x8, at::Tensor W8, at::Tensor C, at::Tensor x_scales, OptTensor w_scales, OptTensor bias, OptTensor residual,
                 const std::string& act) {
  int code;
  if (act == "none") code = FG_ACT_NONE;
  else if (act == "gelu" || act == "gelu_erf") code = FG_ACT_GELU_ERF;
  else if (act == "gelu_tanh") code = FG_ACT_GELU_TANH;
  else if (act == "silu") code = FG_ACT_SILU;
  else if (act == "silu_gate") code = FG_ACT_SILU_GATE;
  else throw std::invalid_argument("fastgate_b200: act must be none, gelu, gelu_tanh, silu or silu_gate");
  check_dense(x8, "activation", at::kChar, -1);
  const int64_t device = x8.get_device();
  check_dense(W8, "weight", at::kChar, device);
  check_dense(C, "output", at::kHalf, device);
  if (x8.dim() != 2 || W8.dim() != 2) throw std::runtime_error("fastgate_b200: activation and weight must be 2-D");
  const int64_t M = x8.size(0), K = x8.size(1), N = W8.size(0);
  if (W8.size(1) != K) throw std::runtime_error("fastgate_b200: activation and weight disagree on K");
  const int64_t width = code == FG_ACT_SILU_GATE ? N / 2 : N;
  if (C.numel() != M * width) throw std::runtime_error("fastgate_b200: output must hold M*N elements (M*N/2 with silu_gate)");
  const bool f32 = x_scales.defined() && x_scales.scalar_type() == at::kFloat;
  check_dense(x_scales, "x_scales", f32 ? at::kFloat : at::kHalf, device);
  if (x_scales.numel() != M) throw std::runtime_error("fastgate_b200: x_scales must hold M elements");
  auto optional_half = [&](const OptTensor& t, const char* name, int64_t n) -> const void* {
    if (!given(t)) return nullptr;
    check_dense(*t, name, at::kHalf, device);
    if (t->numel() != n) throw std::runtime_error(std::string("fastgate_b200: ") + name + " must hold " + std::to_string(n) + " elements");
    return t->data_ptr();
  };
  const void* ws_ptr = optional_half(w_scales, "w_scales", N);
  const void* bias_ptr = optional_half(bias, "bias", N);
  const void* res_ptr = optional_half(residual, "residual", M * width);
  if (M == 0) return;
  if ((N % 128) != 0 || (K % 128) != 0 || N <= 0 || K <= 0)
    throw std::invalid_argument("K(input column) & N(transposed output row) must be multiple of 128!");
  if (K > 131072 - 128) bad_argument("K must be at most 130944: the sums are 32-bit integers");
  if (M > 0x7fffffff || N > 0x7fffffff) bad_argument("too many rows");
  if (overlap(C, x8) || overlap(C, W8) || overlap(C, x_scales) || (given(w_scales) && overlap(C, *w_scales)) || (given(bias) && overlap(C, *bias)) ||
      (given(residual) && overlap(C, *residual) && C.data_ptr() != residual->data_ptr()))
    bad_argument("the output may be the residual itself; otherwise it must not overlap the inputs");
  const c10::cuda::CUDAGuard guard(x8.device());
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(device).stream();
  int* status = linear_status(static_cast<int>(device));
  int st;
  {
    pybind11::gil_scoped_release nogil;
    st = fg_linear_w8a8(static_cast<const int8_t*>(x8.data_ptr()), static_cast<const int8_t*>(W8.data_ptr()), x_scales.data_ptr(), f32, ws_ptr,
                        C.data_ptr(), static_cast<int>(M), static_cast<int>(N), static_cast<int>(K), bias_ptr, res_ptr, code,
                        status, reinterpret_cast<fg_stream_t>(stream));
  }
  check_status(st);
}

// ---- 4-bit key/value cache -----------------------------------------------------------------
// pages [num_pages, kv_heads, page_size * (D + 8)] uint8
void check_pages(const at::Tensor& pages, int64_t page_size, int64_t kv_heads, int64_t d, int64_t device) {
  check_dense(pages, "pages", at::kByte, device);
  if (d != 64 && d != 128) bad_argument("heads of 64 or 128 channels expected");
  if (page_size < 16 || page_size % 16 != 0 || page_size > (1 << 20)) bad_argument("page_size must be a multiple of 16, at most 2^20");
  if (pages.dim() != 3 || pages.size(0) < 1 || pages.size(1) != kv_heads || pages.size(2) != page_size * (d + 8))
    bad_argument("pages must be [num_pages, kv_heads, page_size * (channels + 8)]");
}

void kv_append_int4(at::Tensor k, at::Tensor v, at::Tensor pages, at::Tensor slots, int64_t page_size, OptTensor cos_sin,
                    OptTensor positions, OptTensor q, OptTensor q_out, bool interleaved, OptTensor status) {
  check_rows(k, "k", -1);
  const int64_t device = k.get_device();
  check_rows(v, "v", device);
  if (k.sizes() != v.sizes()) bad_argument("k and v must have one shape");
  const int64_t T = k.size(0), heads = k.size(1), d = k.size(2);
  check_pages(pages, page_size, heads, d, device);
  const int slots64 = check_index(slots, "slots", T, device);
  const float* table = nullptr;
  const void* pos = nullptr;
  int64_t table_len = 0;
  int pos64 = 0;
  if (given(cos_sin) != given(positions)) bad_argument("cos_sin and positions go together");
  if (given(cos_sin)) {
    check_dense(*cos_sin, "cos_sin", at::kFloat, device);
    if (cos_sin->dim() != 2 || cos_sin->size(0) < 1 || cos_sin->size(1) != d) bad_argument("cos_sin must be [positions, channels]: cosines, then sines");
    pos64 = check_index(*positions, "positions", T, device);
    table = cos_sin->data_ptr<float>();
    table_len = cos_sin->size(0);
    pos = positions->data_ptr();
  }
  const void* qp = nullptr;
  void* qo = nullptr;
  int64_t ldq = 0, ldqo = 0, q_heads = 0;
  if (given(q)) {
    if (!given(cos_sin)) bad_argument("q without cos_sin and positions");
    check_rows(*q, "q", device);
    at::Tensor o = given(q_out) ? *q_out : *q;
    check_rows(o, "q_out", device);
    if (q->size(0) != T || q->size(2) != d || q->size(1) < 1 || o.sizes() != q->sizes()) bad_argument("q and q_out must be [tokens, q_heads, channels]");
    if (rows_overlap(o, *q) && !(o.data_ptr() == q->data_ptr() && row_stride(o) == row_stride(*q))) bad_argument("q_out may be q itself, but not overlap it otherwise");
    if (rows_overlap(o, k) || rows_overlap(o, v) || overlap(o, pages) || overlap(o, slots) || overlap(o, *cos_sin) || overlap(o, *positions))
      bad_argument("q_out must not overlap k, v, pages, slots, cos_sin or positions");
    qp = q->data_ptr();
    qo = o.data_ptr();
    ldq = row_stride(*q);
    ldqo = row_stride(o);
    q_heads = q->size(1);
  } else if (given(q_out)) {
    bad_argument("q_out without q");
  }
  if (overlap(pages, k) || overlap(pages, v) || overlap(pages, slots) || (given(q) && overlap(pages, *q)) ||
      (given(cos_sin) && (overlap(pages, *cos_sin) || overlap(pages, *positions))))
    bad_argument("pages must not overlap the other tensors");
  int* sp = status_ptr(status, device);
  if (T == 0 || heads == 0) return;
  if (row_stride(k) % 8 || row_stride(v) % 8 || ldq % 8 || ldqo % 8) bad_argument("token strides must be multiples of 8 elements");
  if (heads > 16384 || q_heads > 16384) bad_argument("too many heads");
  const c10::cuda::CUDAGuard guard(k.device());
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(device).stream();
  int st;
  {
    pybind11::gil_scoped_release nogil;
    st = fg_kv_append_int4(k.data_ptr(), row_stride(k), v.data_ptr(), row_stride(v), T, static_cast<int>(heads), static_cast<int>(d),
                           pages.data_ptr(), pages.size(0), static_cast<int>(page_size), slots.data_ptr(), slots64, table, table_len, pos,
                           pos64, qp, ldq, qo, ldqo, static_cast<int>(q_heads), interleaved, sp, reinterpret_cast<fg_stream_t>(stream));
  }
  check_status(st);
}

void kv_read_int4(at::Tensor pages, at::Tensor slots, at::Tensor k_out, at::Tensor v_out, int64_t page_size, OptTensor status) {
  check_dense(k_out, "k_out", at::kHalf, -1);
  const int64_t device = k_out.get_device();
  check_dense(v_out, "v_out", at::kHalf, device);
  if (k_out.dim() != 3 || k_out.sizes() != v_out.sizes()) bad_argument("k_out and v_out must be [tokens, kv_heads, channels]");
  const int64_t T = k_out.size(0), heads = k_out.size(1), d = k_out.size(2);
  check_pages(pages, page_size, heads, d, device);
  const int slots64 = check_index(slots, "slots", T, device);
  int* sp = status_ptr(status, device);
  if (overlap(k_out, v_out) || overlap(k_out, pages) || overlap(v_out, pages) || overlap(k_out, slots) || overlap(v_out, slots))
    bad_argument("k_out, v_out, pages and slots must not overlap");
  if (T == 0 || heads == 0) return;
  if (heads > 16384) bad_argument("too many heads");
  const c10::cuda::CUDAGuard guard(k_out.device());
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(device).stream();
  int st;
  {
    pybind11::gil_scoped_release nogil;
    st = fg_kv_read_int4(pages.data_ptr(), pages.size(0), static_cast<int>(page_size), static_cast<int>(heads), static_cast<int>(d),
                         slots.data_ptr(), slots64, T, k_out.data_ptr(), v_out.data_ptr(), sp, reinterpret_cast<fg_stream_t>(stream));
  }
  check_status(st);
}

std::mutex g_attn_mu;
std::map<std::pair<int64_t, int64_t>, at::Tensor> g_attn_ws;

struct AttentionWorkspace {
  at::Tensor buf;  // keeps an eager call's memory alive
  void* ptr;
};
// One workspace per (device, stream), made on the first call, or the graph's own while one is captured.
AttentionWorkspace attention_workspace(int64_t device, cudaStream_t stream) {
  const size_t bytes = fg_kv_attention_workspace_bytes();
  if (void* p = graph_workspace(static_cast<int>(device), stream, bytes)) return {at::Tensor(), p};
  std::lock_guard<std::mutex> lk(g_attn_mu);
  at::Tensor& t = g_attn_ws[{device, reinterpret_cast<int64_t>(stream)}];
  if (!t.defined()) {
    at::Tensor made = at::empty({static_cast<int64_t>(bytes)}, at::TensorOptions().dtype(at::kByte).device(at::kCUDA, static_cast<c10::DeviceIndex>(device)));
    check_status(fg_kv_attention_workspace_init(made.data_ptr(), bytes, reinterpret_cast<fg_stream_t>(stream)));
    t = made;
  }
  return {t, t.data_ptr()};
}

void kv_attention_int4(at::Tensor q, at::Tensor pages, at::Tensor block_table, at::Tensor seq_lens, at::Tensor out, int64_t page_size,
                       OptTensor q_starts, c10::optional<double> scale, OptTensor status) {
  check_rows(q, "q", -1);
  const int64_t device = q.get_device();
  check_rows(out, "out", device);
  if (out.sizes() != q.sizes()) bad_argument("out must have the shape of q");
  if (rows_overlap(out, q)) bad_argument("out must not overlap q");
  const int64_t T = q.size(0), q_heads = q.size(1), d = q.size(2);
  check_cuda(pages, "pages", at::kByte, device);
  if (pages.dim() != 3) bad_argument("pages must be [num_pages, kv_heads, page_size * (channels + 8)]");
  const int64_t heads = pages.size(1);
  check_pages(pages, page_size, heads, d, device);
  if (heads < 1 || q_heads < 1 || q_heads % heads != 0) bad_argument("the number of query heads must be a multiple of the number of key/value heads");
  check_cuda(block_table, "block_table", at::kInt, device);
  if (block_table.dim() != 2 || (block_table.size(1) > 1 && block_table.stride(1) != 1)) bad_argument("block_table must be [batch, pages] with dense rows");
  const int64_t B = block_table.size(0), width = block_table.size(1);
  check_dense(seq_lens, "seq_lens", at::kInt, device);
  if (seq_lens.dim() != 1 || seq_lens.size(0) != B) bad_argument("seq_lens must hold one length per sequence");
  const int* starts = nullptr;
  if (given(q_starts)) {
    check_dense(*q_starts, "q_starts", at::kInt, device);
    if (q_starts->dim() != 1 || q_starts->size(0) != B + 1) bad_argument("q_starts must hold batch + 1 row numbers");
    starts = q_starts->data_ptr<int>();
  } else if (T != B) {
    bad_argument("without q_starts there is one row of q per sequence");
  }
  if (overlap(out, pages) || overlap(out, block_table) || overlap(out, seq_lens) || (given(q_starts) && overlap(out, *q_starts)))
    bad_argument("out must not overlap pages, block_table, seq_lens or q_starts");
  int* sp = status_ptr(status, device);
  const double sc = scale.has_value() ? *scale : 1.0 / std::sqrt(static_cast<double>(d));
  if (!(sc > 0) || !(sc <= 1048576.0)) bad_argument("scale must be positive, and at most 2^20");
  if (T == 0 || B == 0) return;
  if (width < 1) bad_argument("block_table must have a column");
  const int64_t ldt = B > 1 ? block_table.stride(0) : width;
  if (ldt < width) bad_argument("rows of block_table overlap");
  if (row_stride(q) % 8 || row_stride(out) % 8) bad_argument("token strides must be multiples of 8 elements");
  if (row_stride(out) < q_heads * d || row_stride(q) < q_heads * d) bad_argument("token strides must be at least q_heads * channels");
  if (B > 0x7fffffff || width > 0x7fffffff || T > 0x7fffffff / q_heads) bad_argument("too many rows");
  const c10::cuda::CUDAGuard guard(q.device());
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(device).stream();
  const AttentionWorkspace ws = attention_workspace(device, stream);
  int st;
  {
    pybind11::gil_scoped_release nogil;
    st = fg_kv_attention_int4(q.data_ptr(), row_stride(q), out.data_ptr(), row_stride(out), T, static_cast<int>(q_heads),
                              static_cast<int>(heads), static_cast<int>(d), pages.data_ptr(), pages.size(0), static_cast<int>(page_size),
                              block_table.data_ptr<int>(), ldt, static_cast<int>(width), seq_lens.data_ptr<int>(), starts,
                              static_cast<int>(B), static_cast<float>(sc), sp, ws.ptr, fg_kv_attention_workspace_bytes(),
                              reinterpret_cast<fg_stream_t>(stream));
  }
  check_status(st);
}

}  // namespace

void bind_serving(pybind11::module& m) {
  namespace py = pybind11;
  m.def("add_rmsnorm", &add_rmsnorm, py::arg("x"), py::arg("weight"), py::arg("out"), py::arg("residual") = py::none(),
        py::arg("eps") = 1e-6, py::arg("scales") = py::none(), py::arg("residual_out") = py::none(),
        "h = x (+ residual); residual_out (default: residual, in place) = h; out = h / sqrt(mean h^2 + eps) * weight.  x [M,K] fp16; "
        "residual fp16 or fp32; out fp16, or int8 with one fp32 scale per row in `scales` (the activations of linear_int8)");
  m.def("linear_int8", &linear_int8, py::arg("x8"), py::arg("W8"), py::arg("C"), py::arg("x_scales"), py::arg("w_scales") = py::none(),
        py::arg("bias") = py::none(), py::arg("residual") = py::none(), py::arg("act") = "none",
        "C[M,N] = act(x8 . W8^T * x_scales[m] * w_scales[n] + bias) + residual: int8 x8 [M,K] (add_rmsnorm, quantize_int8) and W8 [N,K], exact "
        "integer sums; x_scales fp32 or fp16, the rest fp16; act='silu_gate': C[M,N/2] on a weight from prepack_gate_up");
  m.def("kv_append_int4", &kv_append_int4, py::arg("k"), py::arg("v"), py::arg("pages"), py::arg("slots"), py::arg("page_size"),
        py::arg("cos_sin") = py::none(), py::arg("positions") = py::none(), py::arg("q") = py::none(), py::arg("q_out") = py::none(),
        py::arg("interleaved") = false, py::arg("status") = py::none(),
        "Rotates k (and q, into q_out or in place) by the angles of `positions` and writes the rows k[t], v[t] in 4 bits to slots[t] of the "
        "cache (negative: a padding row, left out); k, v [T,kv_heads,D], q [T,q_heads,D] fp16, cos_sin [positions,D] fp32");
  m.def("kv_read_int4", &kv_read_int4, py::arg("pages"), py::arg("slots"), py::arg("k_out"), py::arg("v_out"), py::arg("page_size"),
        py::arg("status") = py::none(), "The cached rows of `slots` as fp16: k_out, v_out [T,kv_heads,D]");
  m.def("kv_attention_int4", &kv_attention_int4, py::arg("q"), py::arg("pages"), py::arg("block_table"), py::arg("seq_lens"), py::arg("out"),
        py::arg("page_size"), py::arg("q_starts") = py::none(), py::arg("scale") = py::none(), py::arg("status") = py::none(),
        "Attention of q [T,q_heads,D] over the 4-bit cache: sequence b sees seq_lens[b] rows in the pages of block_table[b], each of its "
        "query rows (q_starts[b]..q_starts[b+1], default one per sequence, the last rows of the sequence) those up to its own");
}
