// Bindings of serving in block-scaled 8 bits (fp8_rows.cu, fp8_gemm.cu). Shapes and types are looked at before the device, so that a call
// that cannot be answered is refused alike wherever its tensors lie.
#include "binding_helpers.h"
#include "fp8_block.h"

namespace {

using namespace mb_bind;
using OptTensor = c10::optional<at::Tensor>;

constexpr int64_t kBlock = 128;
int64_t blocks(int64_t n) { return (n + kBlock - 1) / kBlock; }
bool aligned16(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

void check_width(int64_t k, const char* name) {
  TORCH_CHECK(k > 0 && k % 16 == 0 && k < (1 << 24), name, ": rows of 8-bit values are a multiple of 16 wide, got ", k);
}
void check_device(const at::Tensor& like, const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device(), name, " must be a CUDA tensor on the device of the other operands");
}
// A bf16 matrix whose rows may be apart; `cols` < 0: any.
void check_bf16_rows(const at::Tensor& t, int64_t rows, int64_t cols, const char* name) {
  TORCH_CHECK(t.scalar_type() == at::kBFloat16 && t.dim() == 2 && (t.size(1) <= 1 || t.stride(1) == 1), name,
              " must be a bf16 matrix with contiguous rows");
  TORCH_CHECK((rows < 0 || t.size(0) == rows) && (cols < 0 || t.size(1) == cols), name, " must be a CUDA tensor [", rows, ", ", cols, "], got [",
              t.size(0), ", ", t.size(1), "]");
  TORCH_CHECK(t.size(0) <= 1 || t.stride(0) >= t.size(1), name, ": rows must not overlap");
}
void check_vectors(const at::Tensor& t, const char* name) {
  TORCH_CHECK(aligned16(t) && (t.size(0) <= 1 || t.stride(0) % 8 == 0), name, " needs 16-byte aligned rows");
}
long long pitch(const at::Tensor& t) { return t.size(0) <= 1 ? t.size(1) : t.stride(0); }

void check_rows(const at::Tensor& q, const at::Tensor& s) {
  TORCH_CHECK(q.scalar_type() == at::kFloat8_e4m3fn && q.dim() == 2 && (q.size(1) <= 1 || q.stride(1) == 1), "x: 8-bit rows are a float8_e4m3fn matrix with contiguous rows");
  check_width(q.size(1), "x");
  TORCH_CHECK(q.size(0) <= 1 || (q.stride(0) >= q.size(1) && q.stride(0) % 16 == 0), "x needs rows that are a multiple of 16 bytes apart");
  TORCH_CHECK(s.scalar_type() == at::kFloat && s.is_contiguous() && s.dim() == 2 && s.size(0) == q.size(0) && s.size(1) == blocks(q.size(1)),
              "x: scales must be contiguous fp32 [", q.size(0), ", ", blocks(q.size(1)), "]");
  TORCH_CHECK(q.size(0) <= (1ll << 31) - 256, "x: at most 2^31 - 256 rows, which whole tiles of 256 reach in 32 bits, got ", q.size(0));
}

std::pair<at::Tensor, at::Tensor> new_rows(int64_t rows, int64_t cols, const at::Tensor& like) {
  return {at::empty({rows, cols}, like.options().dtype(at::kFloat8_e4m3fn)), at::empty({rows, blocks(cols)}, like.options().dtype(at::kFloat))};
}
void check_launch(cudaError_t e, const char* name) {
  if (e != cudaSuccess) cudaGetLastError();  // (reported here)
  TORCH_CHECK(e == cudaSuccess, name, ": ", cudaGetErrorString(e));
}

// x bf16 [T, K] -> (q e4m3 [T, K], scales fp32 [T, ceil(K / 128)])
std::tuple<at::Tensor, at::Tensor> fp8_quantize_rows(const at::Tensor& x) {
  check_bf16_rows(x, -1, -1, "x");
  check_width(x.size(1), "x");
  check_device(x, x, "x");
  check_vectors(x, "x");
  const c10::cuda::CUDAGuard guard(x.device());
  auto [q, s] = new_rows(x.size(0), x.size(1), x);
  check_launch(mb::fp8_quantize_rows(x.data_ptr(), pitch(x), x.size(0), static_cast<int>(x.size(1)), static_cast<uint8_t*>(q.data_ptr()), s.data_ptr<float>(),
                                     cur_stream()), "fp8_quantize_rows");
  return {q, s};
}

// -> (q, scales, x + residual in bf16 or x itself without a residual, the normalised rows in bf16 if kept)
std::tuple<at::Tensor, at::Tensor, at::Tensor, OptTensor> fp8_rmsnorm_rows(const at::Tensor& x, const at::Tensor& w, double eps, const OptTensor& residual,
                                                                           bool keep) {
  check_bf16_rows(x, -1, -1, "x");
  const int64_t T = x.size(0), H = x.size(1);
  check_width(H, "x");
  TORCH_CHECK(H <= 32768, "x: rows of at most 32768 columns are normalised, got ", H);
  TORCH_CHECK(w.scalar_type() == at::kBFloat16 && w.is_contiguous() && w.dim() == 1 && w.size(0) == H, "weight must be contiguous bf16 [", H, "]");
  if (residual.has_value()) check_bf16_rows(*residual, T, H, "residual");
  check_device(x, x, "x");
  check_device(x, w, "weight");
  check_vectors(x, "x");
  TORCH_CHECK(aligned16(w), "weight must be 16-byte aligned");
  if (residual.has_value()) {
    check_device(x, *residual, "residual");
    check_vectors(*residual, "residual");
  }
  const c10::cuda::CUDAGuard guard(x.device());
  auto [q, s] = new_rows(T, H, x);
  at::Tensor sum = residual.has_value() ? at::empty({T, H}, x.options()) : x;
  OptTensor y;
  if (keep) y = at::empty({T, H}, x.options());
  check_launch(mb::fp8_rmsnorm_rows(x.data_ptr(), pitch(x), residual.has_value() ? residual->data_ptr() : nullptr, residual.has_value() ? pitch(*residual) : 0,
                                    w.data_ptr(), static_cast<float>(eps), T, static_cast<int>(H), static_cast<uint8_t*>(q.data_ptr()), s.data_ptr<float>(),
                                    residual.has_value() ? sum.data_ptr() : nullptr, keep ? y->data_ptr() : nullptr, cur_stream()), "fp8_rmsnorm_rows");
  return {q, s, sum, y};
}

// q, scales of T tokens -> those of `src.numel()` rows in expert order (rows past the live ones are left unwritten)
std::tuple<at::Tensor, at::Tensor> fp8_permute_rows(const at::Tensor& q, const at::Tensor& s, const at::Tensor& src, const at::Tensor& num_tiles, int64_t top_k) {
  check_rows(q, s);
  TORCH_CHECK(q.is_contiguous(), "x must be contiguous");
  TORCH_CHECK(src.scalar_type() == at::kInt && src.is_contiguous() && src.dim() == 1, "src must be contiguous int32 [rows]");
  TORCH_CHECK(num_tiles.scalar_type() == at::kInt && num_tiles.is_contiguous() && num_tiles.numel() >= 2, "num_tiles must be int32 {live tiles, live rows}");
  TORCH_CHECK(top_k >= 1 && top_k < (1 << 16), "top_k must be positive");
  check_device(q, q, "x");
  check_device(q, s, "x's scales");
  check_device(q, src, "src");
  check_device(q, num_tiles, "num_tiles");
  TORCH_CHECK(aligned16(q), "x needs 16-byte aligned rows");
  const c10::cuda::CUDAGuard guard(q.device());
  auto [pq, ps] = new_rows(src.numel(), q.size(1), q);
  check_launch(mb::fp8_permute_rows(static_cast<const uint8_t*>(q.data_ptr()), s.data_ptr<float>(), src.data_ptr<int>(), num_tiles.data_ptr<int>(),
                                    static_cast<int>(top_k), src.numel(), q.size(0), static_cast<int>(q.size(1)), static_cast<uint8_t*>(pq.data_ptr()),
                                    ps.data_ptr<float>(), cur_stream()), "fp8_permute_rows");
  return {pq, ps};
}

// The parts of a product: x, W [N, K] or [groups, N, K], the row tiles of a grouped one, and what an ungated one adds to and writes.
mb::Fp8Gemm product(const at::Tensor& xq, const at::Tensor& xs, const at::Tensor& wq, const at::Tensor& ws, bool gated, int64_t halves, const OptTensor& tile_group,
                    const OptTensor& num_tiles, const OptTensor& status, const OptTensor& residual = {}, const OptTensor& out = {}) {
  check_rows(xq, xs);
  const bool grouped = tile_group.has_value();
  TORCH_CHECK(grouped == num_tiles.has_value(), "tile_group and num_tiles are given together");
  TORCH_CHECK(wq.scalar_type() == at::kFloat8_e4m3fn && wq.is_contiguous() && wq.dim() == (grouped ? 3 : 2), "weight must be contiguous float8_e4m3fn ",
              grouped ? "[experts, N, K]" : "[N, K]");
  mb::Fp8Gemm p{};
  p.groups = grouped ? wq.size(0) : 1;
  const int64_t N = wq.size(-2), K = wq.size(-1);
  TORCH_CHECK(K == xq.size(1), "x is ", xq.size(1), " wide, the weight ", K);
  TORCH_CHECK(p.groups >= 1 && N >= 1 && N < (1 << 24) && p.groups * N < (1ll << 31) - 256, "weight: sizes out of range");
  TORCH_CHECK(halves == 1 || (halves == 2 && N % 2 == 0), "weight: halves is 1, or 2 for a gate-up weight of an even number of rows");
  if (gated) {
    TORCH_CHECK(N % 2 == 0, "a gate-up weight has an even number of rows");
    check_width(N / 2, "gate");
  }
  // halves that are a multiple of 128 rows have the same blocks either way
  TORCH_CHECK(gated == (halves == 2) || (N % 2 == 0 && (N / 2) % kBlock == 0), "weight: its blocks are those of ", halves == 2 ? "a gate-up weight" : "one matrix",
              ", this product reads ", gated ? "a gate-up weight (halves = 2)" : "one matrix (halves = 1)");
  const int64_t bn = gated ? 2 * blocks(N / 2) : blocks(N);
  TORCH_CHECK(ws.scalar_type() == at::kFloat && ws.is_contiguous() && ws.dim() == wq.dim() && ws.size(-2) == bn && ws.size(-1) == blocks(K) &&
                  (!grouped || ws.size(0) == wq.size(0)),
              "weight: scales must be contiguous fp32 [", grouped ? "experts, " : "", bn, ", ", blocks(K), "]");
  if (grouped) {
    TORCH_CHECK(tile_group->scalar_type() == at::kInt && tile_group->is_contiguous() && tile_group->dim() == 2 && tile_group->size(1) == 4,
                "tile_group must be contiguous int32 [tiles, 4]");
    TORCH_CHECK(num_tiles->scalar_type() == at::kInt && num_tiles->numel() >= 1, "num_tiles must be int32");
    TORCH_CHECK(tile_group->size(0) < (1 << 24), "tile_group: too many tiles");
  }
  if (status.has_value()) TORCH_CHECK(status->scalar_type() == at::kInt && status->numel() >= 1, "status must be int32");
  if (residual.has_value()) check_bf16_rows(*residual, xq.size(0), N, "residual");
  if (out.has_value()) check_bf16_rows(*out, xq.size(0), N, "out");
  check_device(xq, xq, "x");
  check_device(xq, xs, "x's scales");
  check_device(xq, wq, "weight");
  check_device(xq, ws, "weight's scales");
  TORCH_CHECK(aligned16(xq) && aligned16(wq), "8-bit operands must be 16-byte aligned");
  if (grouped) {
    check_device(xq, *tile_group, "tile_group");
    check_device(xq, *num_tiles, "num_tiles");
    TORCH_CHECK(aligned16(*tile_group), "tile_group must be 16-byte aligned");
    p.tile_group = tile_group->data_ptr<int>();
    p.num_tiles = num_tiles->data_ptr<int>();
    p.max_tiles = static_cast<int>(tile_group->size(0));
  }
  if (status.has_value()) {
    check_device(xq, *status, "status");
    p.status = status->data_ptr<int>();
  }
  if (residual.has_value()) {
    check_device(xq, *residual, "residual");
    p.residual = residual->data_ptr();
    p.ldr = pitch(*residual);
  }
  if (out.has_value()) check_device(xq, *out, "out");
  p.M = static_cast<int>(xq.size(0));
  p.N = static_cast<int>(N);
  p.K = static_cast<int>(K);
  p.x = static_cast<const uint8_t*>(xq.data_ptr());
  p.ldx = pitch(xq);
  p.xs = xs.data_ptr<float>();
  p.w = static_cast<const uint8_t*>(wq.data_ptr());
  p.ws = ws.data_ptr<float>();
  return p;
}

// Launches with a workspace of the allocator's, which a captured graph keeps to itself.
void launch(mb::Fp8Gemm& p, const at::Tensor& like, const char* name) {
  at::Tensor ws;
  if (const long long bytes = mb::fp8_gemm_workspace(p)) {
    ws = at::empty({bytes}, like.options().dtype(at::kByte));
    p.workspace = ws.data_ptr();
  }
  TORCH_CHECK(mb::fp8_gemm_launch(p, cur_stream()) == 0, name, ": ", mb::fp8_last_error());
}

at::Tensor fp8_linear(const at::Tensor& xq, const at::Tensor& xs, const at::Tensor& wq, const at::Tensor& ws, int64_t halves, const OptTensor& residual,
                      const OptTensor& tile_group, const OptTensor& num_tiles, const OptTensor& out, const OptTensor& status) {
  mb::Fp8Gemm p = product(xq, xs, wq, ws, false, halves, tile_group, num_tiles, status, residual, out);
  const c10::cuda::CUDAGuard guard(xq.device());
  at::Tensor y = out.has_value() ? *out : at::empty({p.M, p.N}, xs.options().dtype(at::kBFloat16));
  p.y = y.data_ptr();
  p.ldy = pitch(y);
  launch(p, xs, "fp8_linear");
  return y;
}

std::tuple<at::Tensor, at::Tensor> fp8_gated_linear(const at::Tensor& xq, const at::Tensor& xs, const at::Tensor& wq, const at::Tensor& ws, int64_t halves,
                                                    const OptTensor& tile_group, const OptTensor& num_tiles, const OptTensor& status) {
  mb::Fp8Gemm p = product(xq, xs, wq, ws, true, halves, tile_group, num_tiles, status);
  const c10::cuda::CUDAGuard guard(xq.device());
  auto [q, s] = new_rows(p.M, p.N / 2, xq);
  p.q = static_cast<uint8_t*>(q.data_ptr());
  p.s = s.data_ptr<float>();
  launch(p, xs, "fp8_gated_linear");
  return {q, s};
}

}  // namespace

void register_fp8_block(pybind11::module_& m) {
  namespace py = pybind11;
  m.def("fp8_quantize_rows", &fp8_quantize_rows, py::arg("x"));
  m.def("fp8_rmsnorm_rows", &fp8_rmsnorm_rows, py::arg("x"), py::arg("weight"), py::arg("eps"), py::arg("residual") = py::none(), py::arg("keep") = false);
  m.def("fp8_permute_rows", &fp8_permute_rows, py::arg("q"), py::arg("scales"), py::arg("src"), py::arg("num_tiles"), py::arg("top_k"));
  m.def("fp8_linear", &fp8_linear, py::arg("xq"), py::arg("xs"), py::arg("wq"), py::arg("ws"), py::arg("halves"), py::arg("residual") = py::none(),
        py::arg("tile_group") = py::none(), py::arg("num_tiles") = py::none(), py::arg("out") = py::none(), py::arg("status") = py::none());
  m.def("fp8_grouped_launches", &mb::fp8_grouped_launches, py::arg("rows"), py::arg("experts"), py::arg("n"), py::arg("k"), py::arg("gated"), py::arg("tiles"));
  m.def("fp8_gated_linear", &fp8_gated_linear, py::arg("xq"), py::arg("xs"), py::arg("wq"), py::arg("ws"), py::arg("halves"), py::arg("tile_group") = py::none(),
        py::arg("num_tiles") = py::none(), py::arg("status") = py::none());
}
