// Torch bridge: torch.ops.vecops_b200.matmul / matmul_out / sdpa and the decode-step operators (quantize_blocks,
// matmul_f8_blocks, cache_append, sdpa_shared_prefix) hand CUDA tensors straight to the operator bridge or the C ABI
// (vecops_operator_bridge_invoke_v1) on the current stream - dispatcher to C++ to kernel, no Python on the hot path.
// It stands where vecops' generated Torch adapters stand (python/vecops/ops/torch.py `register` -> generated bridge
// DSO -> vecops_operator_bridge_invoke_v1, include/vecops/runtime/OperatorBridgeAbi.h:156-158).
//
// torch is plumbing here (tensors, the caching allocator for scratch, the current stream); all arithmetic is in the
// library's own kernels.  Calls are enqueued asynchronously, like any torch CUDA op.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/library.h>

#include <array>
#include <string>
#include <tuple>
#include <utility>
#include <vector>

#include "vecops_b200/decode_cuda.h"
#include "vecops_b200/matmul_cuda.h"
#include "vecops_b200/operator_bridge.h"

namespace {

uint32_t dtype_code(at::ScalarType type) {
  switch (type) {
    case at::kFloat: return VECOPS_DTYPE_F32;
    case at::kBFloat16: return VECOPS_DTYPE_BF16;
    case at::kHalf: return VECOPS_DTYPE_F16;
    case at::kChar: return VECOPS_DTYPE_I8;
    case at::kByte: return VECOPS_DTYPE_U8;
    case at::kInt: return VECOPS_DTYPE_I32;
    default: TORCH_CHECK(false, "vecops_b200: dtype ", type, " has no vecops code on this path");
  }
}

struct ErrorText {
  std::array<char, 512> text{};
  VecopsError record{};
  ErrorText() {
    record.struct_size = sizeof(VecopsError);
    record.message = text.data();
    record.message_capacity = text.size();
  }
  void check(int32_t code, const char* what) const { TORCH_CHECK(code == VECOPS_STATUS_OK, "vecops_b200 ", what, " failed (", code, "): ", text.data()); }
};

VecopsValue tensor_value(const at::Tensor& t, bool writable) {
  VecopsValue v{};
  v.struct_size = sizeof(VecopsValue);
  v.kind = VECOPS_VALUE_TENSOR;
  VecopsTensorView& view = v.value.tensor;
  view.struct_size = sizeof(VecopsTensorView);
  view.data = t.data_ptr();
  view.byte_offset = 0;
  view.device_type = t.is_cuda() ? VECOPS_DEVICE_CUDA : VECOPS_DEVICE_CPU;
  view.device_index = t.is_cuda() ? static_cast<int32_t>(t.get_device()) : 0;
  view.dtype = dtype_code(t.scalar_type());
  view.rank = static_cast<uint32_t>(t.dim());
  view.sizes = t.sizes().data();      // owned by the tensor, which outlives the call
  view.strides = t.strides().data();
  view.flags = VECOPS_TENSOR_READ | (writable ? VECOPS_TENSOR_WRITE : 0);
  return v;
}

VecopsValue none_value() {
  VecopsValue v{};
  v.struct_size = sizeof(VecopsValue);
  v.kind = VECOPS_VALUE_NONE;
  return v;
}

VecopsValue scalar_value(uint32_t dtype, double real, int64_t integer) {
  VecopsValue v{};
  v.struct_size = sizeof(VecopsValue);
  v.kind = VECOPS_VALUE_SCALAR;
  v.value.scalar.struct_size = sizeof(VecopsScalar);
  v.value.scalar.dtype = dtype;
  if (dtype == VECOPS_DTYPE_F32) v.value.scalar.value.f64 = real;  // scalars travel widened, the tag says what they were
  else v.value.scalar.value.i64 = integer;
  return v;
}

// c = activation((cin + a . b_nk^T) * alpha * column_scale), written into `c`
void matmul_out(const at::Tensor& a, const at::Tensor& b_nk, at::Tensor& c, const c10::optional<at::Tensor>& column_scale,
                const c10::optional<at::Tensor>& cin, double alpha, int64_t activation, double clamp_lo, double clamp_hi,
                const c10::optional<at::Tensor>& row_scale) {
  TORCH_CHECK(a.is_cuda() && b_nk.is_cuda() && c.is_cuda(), "vecops_b200.matmul: CUDA tensors only (there is no CPU path)");
  TORCH_CHECK(a.dim() == 2 && b_nk.dim() == 2 && c.dim() == 2, "vecops_b200.matmul: a [M,K], b_nk [N,K], c [M,N]");
  const c10::cuda::CUDAGuard guard(c.device());
  const bool has_scale = column_scale.has_value() && column_scale->defined();
  const bool has_cin = cin.has_value() && cin->defined();
  at::Tensor cin_view;
  if (has_cin) cin_view = cin->expand({c.size(0), c.size(1)});  // a bias row or a column becomes a stride-0 view
  std::vector<VecopsValue> values{tensor_value(a, false), tensor_value(b_nk, false), tensor_value(c, true)};
  const bool has_row = row_scale.has_value() && row_scale->defined();
  const bool fused = has_cin || alpha != 1.0 || activation != 0 || has_row;
  if (has_scale || fused) values.push_back(has_scale ? tensor_value(*column_scale, false) : none_value());
  if (fused) {
    values.push_back(has_cin ? tensor_value(cin_view, false) : none_value());
    values.push_back(scalar_value(VECOPS_DTYPE_F32, alpha, 0));
    values.push_back(scalar_value(VECOPS_DTYPE_I32, 0.0, activation));
    values.push_back(scalar_value(VECOPS_DTYPE_F32, clamp_lo, 0));
    values.push_back(scalar_value(VECOPS_DTYPE_F32, clamp_hi, 0));
    if (has_row) values.push_back(tensor_value(*row_scale, false));
  }
  VecopsExecutionContext context{};
  context.struct_size = sizeof(VecopsExecutionContext);
  context.stream = at::cuda::getCurrentCUDAStream(c.get_device()).stream();
  context.flags = VECOPS_B200_CONTEXT_FLAG_ASYNC;
  VecopsCall call{};
  call.struct_size = sizeof(VecopsCall);
  call.num_values = static_cast<uint32_t>(values.size());
  call.values = values.data();
  call.context = &context;
  const uint64_t handle = vecops_b200_matmul_operator();
  ErrorText error;
  uint64_t need = 0;
  error.check(vecops_b200_operator_workspace(handle, &call, &need, &error.record), "workspace query");
  at::Tensor scratch;  // from torch's caching allocator: freed blocks are re-issued only to later work on this stream
  if (need != 0) {
    scratch = at::empty({static_cast<int64_t>(need)}, a.options().dtype(at::kByte));
    call.workspace = scratch.data_ptr();
    call.workspace_size = need;
  }
  error.check(vecops_operator_bridge_invoke_v1(handle, &call, 0, nullptr, &error.record), "matmul");
}

at::Tensor matmul(const at::Tensor& a, const at::Tensor& b_nk, const c10::optional<at::Tensor>& column_scale,
                  const c10::optional<at::Tensor>& cin, double alpha, int64_t activation, double clamp_lo, double clamp_hi,
                  c10::optional<at::ScalarType> out_dtype, const c10::optional<at::Tensor>& row_scale) {
  TORCH_CHECK(a.dim() == 2 && b_nk.dim() == 2, "vecops_b200.matmul: a [M,K], b_nk [N,K]");
  at::ScalarType type = a.scalar_type();
  if (out_dtype.has_value()) type = *out_dtype;
  else if (a.scalar_type() == at::kChar || a.scalar_type() == at::kByte) type = at::kInt;  // 8-bit operands accumulate in int32
  at::Tensor c = at::empty({a.size(0), b_nk.size(0)}, a.options().dtype(type));
  matmul_out(a, b_nk, c, column_scale, cin, alpha, activation, clamp_lo, clamp_hi, row_scale);
  return c;
}

// Scaled dot-product attention, q [H,Lq,D] | [Lq,D] (k, v likewise), bf16; masks uint8 / bool (non-zero keeps).
at::Tensor sdpa(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, double scale, int64_t causal,
                const c10::optional<at::Tensor>& key_mask, const c10::optional<at::Tensor>& bias, c10::optional<at::ScalarType> out_dtype) {
  TORCH_CHECK(q.is_cuda() && k.is_cuda() && v.is_cuda(), "vecops_b200.sdpa: CUDA tensors only");
  TORCH_CHECK(q.dim() == k.dim() && q.dim() == v.dim() && (q.dim() == 2 || q.dim() == 3), "vecops_b200.sdpa: q, k, v are [L,D] or [H,L,D]");
  const c10::cuda::CUDAGuard guard(q.device());
  const bool heads = q.dim() == 3;
  const int64_t h = heads ? q.size(0) : 1;
  auto dim = [&](const at::Tensor& t, int i) { return t.size(heads ? i + 1 : i); };
  auto stride = [&](const at::Tensor& t, int i) { return t.stride(heads ? i + 1 : i); };
  TORCH_CHECK(!heads || (k.size(0) == h && v.size(0) == h), "vecops_b200.sdpa: head counts disagree (expand shared K / V to the head count)");
  std::vector<int64_t> shape = heads ? std::vector<int64_t>{h, dim(q, 0), dim(v, 1)} : std::vector<int64_t>{dim(q, 0), dim(v, 1)};
  at::Tensor out = at::empty(shape, q.options().dtype(out_dtype.has_value() ? *out_dtype : q.scalar_type()));
  VecopsB200Attention a{};
  a.struct_size = sizeof(VecopsB200Attention);
  a.causal = static_cast<uint32_t>(causal);
  a.lq = dim(q, 0), a.dqk = dim(q, 1), a.lkv = dim(v, 0), a.dv = dim(v, 1);
  TORCH_CHECK(dim(k, 0) == a.lkv && dim(k, 1) == a.dqk, "vecops_b200.sdpa: k must be [Lkv, Dqk]");
  a.q = q.data_ptr(), a.q_stride_row = stride(q, 0), a.q_stride_col = stride(q, 1);
  a.k = k.data_ptr(), a.k_stride_row = stride(k, 0), a.k_stride_col = stride(k, 1);
  a.v = v.data_ptr(), a.v_stride_row = stride(v, 0), a.v_stride_col = stride(v, 1);
  a.out = out.data_ptr(), a.out_stride_row = stride(out, 0), a.out_stride_col = stride(out, 1);
  a.qkv_dtype = dtype_code(q.scalar_type());
  a.out_dtype = dtype_code(out.scalar_type());
  at::Tensor mask_bytes, bias_view;
  if (key_mask.has_value() && key_mask->defined()) {
    mask_bytes = key_mask->to(at::kByte).contiguous();
    TORCH_CHECK(mask_bytes.dim() == 1 && mask_bytes.size(0) == a.lkv, "vecops_b200.sdpa: key_mask is [Lkv]");
    a.key_mask = static_cast<const uint8_t*>(mask_bytes.data_ptr());
  }
  if (bias.has_value() && bias->defined()) {
    TORCH_CHECK(bias->scalar_type() == at::kFloat, "vecops_b200.sdpa: bias is float32");
    bias_view = heads ? bias->expand({h, a.lq, a.lkv}) : bias->expand({a.lq, a.lkv});
    a.bias = static_cast<const float*>(bias_view.data_ptr());
    a.bias_stride_row = stride(bias_view, 0), a.bias_stride_col = stride(bias_view, 1);
    if (heads) a.bias_stride_head = bias_view.stride(0);
  }
  if (heads) {
    a.heads = h;
    a.q_stride_head = q.stride(0), a.k_stride_head = k.stride(0), a.v_stride_head = v.stride(0), a.out_stride_head = out.stride(0);
  }
  a.scale = static_cast<float>(scale);
  a.flags = VECOPS_B200_MATMUL_FLAG_ASYNC;
  a.stream = at::cuda::getCurrentCUDAStream(q.get_device()).stream();
  a.device_index = static_cast<int32_t>(q.get_device());
  ErrorText error;
  uint64_t need = 0;
  error.check(vecops_b200_sdpa_workspace(&a, &need, &error.record), "sdpa workspace query");
  at::Tensor scratch = at::empty({static_cast<int64_t>(need) + 256}, q.options().dtype(at::kByte));
  const uintptr_t base = reinterpret_cast<uintptr_t>(scratch.data_ptr());
  a.workspace = reinterpret_cast<void*>((base + 255) & ~static_cast<uintptr_t>(255));
  a.workspace_size = need;
  error.check(vecops_b200_sdpa_run(&a, &error.record), "sdpa");
  return out;
}

// ---------------------------------------------------------------- the decode step (decode_cuda.h)

void* current_stream(const at::Tensor& t) { return at::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

// `t` is a CUDA tensor on the device of `like`, of the given rank and type.
void check_operand(const at::Tensor& t, const at::Tensor& like, int64_t rank, at::ScalarType type, const char* op, const char* name) {
  TORCH_CHECK(t.is_cuda(), "vecops_b200.", op, ": ", name, " must be a CUDA tensor (there is no CPU path)");
  TORCH_CHECK(t.get_device() == like.get_device(), "vecops_b200.", op, ": ", name, " is on another device than the first operand");
  TORCH_CHECK(t.dim() == rank, "vecops_b200.", op, ": ", name, " must have ", rank, " dimensions, not ", t.dim());
  TORCH_CHECK(t.scalar_type() == type, "vecops_b200.", op, ": ", name, " must be ", type, ", not ", t.scalar_type());
}

void check_rows(const at::Tensor& t, const char* op, const char* name) {
  TORCH_CHECK(t.size(-1) <= 1 || t.stride(-1) == 1, "vecops_b200.", op, ": ", name, " must be contiguous along its last dimension");
}

// x [M,K] -> (e4m3 [M,K] on a row pitch of a multiple of 16, f32 scales [ceil(M / block_rows), ceil(K / 128)])
std::tuple<at::Tensor, at::Tensor> quantize_blocks(const at::Tensor& x, int64_t block_rows) {
  TORCH_CHECK(block_rows == 1 || block_rows == 128, "vecops_b200.quantize_blocks: block_rows is 1 or 128, not ", block_rows);
  TORCH_CHECK(x.is_cuda(), "vecops_b200.quantize_blocks: CUDA tensors only (there is no CPU path)");
  TORCH_CHECK(x.dim() == 2, "vecops_b200.quantize_blocks: x is [M,K]");
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t m = x.size(0), k = x.size(1), pitch = (k + 15) / 16 * 16;
  at::Tensor q = at::empty({m, pitch}, x.options().dtype(at::kFloat8_e4m3fn));
  if (pitch != k) q = q.narrow(1, 0, k);
  at::Tensor scale = at::empty({(m + block_rows - 1) / block_rows, (k + 127) / 128}, x.options().dtype(at::kFloat));
  VecopsB200QuantizeBlocks r{};
  r.struct_size = sizeof(r);
  r.block_rows = static_cast<uint32_t>(block_rows);
  r.rows = m, r.cols = k;
  r.src = x.data_ptr(), r.src_stride_row = x.stride(0), r.src_stride_col = x.stride(1);
  r.src_dtype = dtype_code(x.scalar_type());
  r.flags = VECOPS_B200_MATMUL_FLAG_ASYNC;
  r.dst = q.data_ptr(), r.dst_stride_row = pitch;
  r.scale = scale.data_ptr<float>(), r.scale_stride_row = scale.stride(0), r.scale_stride_col = scale.stride(1);
  r.stream = current_stream(x);
  r.device_index = static_cast<int32_t>(x.get_device());
  ErrorText error;
  error.check(vecops_b200_quantize_blocks(&r, &error.record), "quantize_blocks");
  return {q, scale};
}

// C[M,N] = sum over 128-blocks of K of a_scale * b_scale * (A_block . B_block^T)
at::Tensor matmul_f8_blocks(const at::Tensor& a, const at::Tensor& a_scale, const at::Tensor& b_nk, const at::Tensor& b_scale,
                            c10::optional<at::ScalarType> out_dtype) {
  constexpr const char* op = "matmul_f8_blocks";
  check_operand(a, a, 2, at::kFloat8_e4m3fn, op, "a");
  check_operand(b_nk, a, 2, at::kFloat8_e4m3fn, op, "b_nk");
  check_operand(a_scale, a, 2, at::kFloat, op, "a_scale");
  check_operand(b_scale, a, 2, at::kFloat, op, "b_scale");
  const int64_t m = a.size(0), k = a.size(1), n = b_nk.size(0), blocks = (k + 127) / 128;
  TORCH_CHECK(b_nk.size(1) == k, "vecops_b200.matmul_f8_blocks: a is [M,", k, "], b_nk [N,", b_nk.size(1), "]");
  TORCH_CHECK(a_scale.size(0) == m && a_scale.size(1) == blocks, "vecops_b200.matmul_f8_blocks: a_scale must be [", m, ",", blocks, "]");
  TORCH_CHECK(b_scale.size(0) == (n + 127) / 128 && b_scale.size(1) == blocks, "vecops_b200.matmul_f8_blocks: b_scale must be [", (n + 127) / 128, ",",
              blocks, "]");
  const c10::cuda::CUDAGuard guard(a.device());
  at::Tensor c = at::empty({m, n}, a.options().dtype(out_dtype.has_value() ? *out_dtype : at::kBFloat16));
  VecopsB200MatmulF8 r{};
  r.struct_size = sizeof(r);
  r.m = m, r.n = n, r.k = k;
  r.a = a.data_ptr(), r.a_stride_m = a.stride(0), r.a_stride_k = a.stride(1);
  r.b = b_nk.data_ptr(), r.b_stride_n = b_nk.stride(0), r.b_stride_k = b_nk.stride(1);
  r.a_scale = a_scale.data_ptr<float>(), r.a_scale_stride_m = a_scale.stride(0), r.a_scale_stride_k = a_scale.stride(1);
  r.b_scale = b_scale.data_ptr<float>(), r.b_scale_stride_n = b_scale.stride(0), r.b_scale_stride_k = b_scale.stride(1);
  r.c = c.data_ptr(), r.c_stride_m = c.stride(0), r.c_stride_n = c.stride(1);
  r.c_dtype = dtype_code(c.scalar_type());
  r.flags = VECOPS_B200_MATMUL_FLAG_ASYNC;
  r.stream = current_stream(a);
  r.device_index = static_cast<int32_t>(a.get_device());
  ErrorText error;
  error.check(vecops_b200_matmul_f8_run(&r, &error.record), "matmul_f8_blocks");
  return c;
}

// q [T,Hq,D], k and v [T,Hkv,D] into k_cache, v_cache [pages,page_size,Hkv,D] at slots [T]; returns the rotated q
at::Tensor cache_append(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, at::Tensor k_cache, at::Tensor v_cache, const at::Tensor& slots,
                        const at::Tensor& positions, const at::Tensor& cos_sin, bool interleaved) {
  constexpr const char* op = "cache_append";
  check_operand(q, q, 3, q.scalar_type(), op, "q");
  check_operand(k, q, 3, q.scalar_type(), op, "k");
  check_operand(v, q, 3, q.scalar_type(), op, "v");
  check_operand(k_cache, q, 4, q.scalar_type(), op, "k_cache");
  check_operand(v_cache, q, 4, q.scalar_type(), op, "v_cache");
  check_operand(slots, q, 1, at::kLong, op, "slots");
  check_operand(positions, q, 1, at::kLong, op, "positions");
  check_operand(cos_sin, q, 2, at::kFloat, op, "cos_sin");
  const int64_t t = q.size(0), d = q.size(2), hkv = k.size(1);
  TORCH_CHECK(k.size(0) == t && k.size(2) == d && v.sizes() == k.sizes(), "vecops_b200.cache_append: q is [T,Hq,D], k and v are [T,Hkv,D]");
  TORCH_CHECK(k_cache.size(2) == hkv && k_cache.size(3) == d && v_cache.sizes() == k_cache.sizes(),
              "vecops_b200.cache_append: k_cache and v_cache are [pages,page_size,", hkv, ",", d, "]");
  TORCH_CHECK(slots.size(0) == t && positions.size(0) == t, "vecops_b200.cache_append: slots and positions are [T]");
  TORCH_CHECK(slots.is_contiguous() && positions.is_contiguous(), "vecops_b200.cache_append: slots and positions must be contiguous");
  TORCH_CHECK(cos_sin.size(1) <= d && cos_sin.size(1) % 2 == 0, "vecops_b200.cache_append: cos_sin is [positions,R] with R even and at most ", d);
  for (const auto& [tensor, name] : {std::pair<const at::Tensor&, const char*>{q, "q"}, {k, "k"}, {v, "v"}, {k_cache, "k_cache"}, {v_cache, "v_cache"},
                                     {cos_sin, "cos_sin"}})
    check_rows(tensor, op, name);
  const c10::cuda::CUDAGuard guard(q.device());
  at::Tensor q_out = at::empty(q.sizes(), q.options());
  VecopsB200CacheAppend r{};
  r.struct_size = sizeof(r);
  r.dtype = dtype_code(q.scalar_type());
  r.tokens = t, r.q_heads = q.size(1), r.kv_heads = hkv, r.head_dim = d;
  r.q = q.data_ptr(), r.q_stride_token = q.stride(0), r.q_stride_head = q.stride(1);
  r.k = k.data_ptr(), r.k_stride_token = k.stride(0), r.k_stride_head = k.stride(1);
  r.v = v.data_ptr(), r.v_stride_token = v.stride(0), r.v_stride_head = v.stride(1);
  r.q_out = q_out.data_ptr(), r.q_out_stride_token = q_out.stride(0), r.q_out_stride_head = q_out.stride(1);
  r.k_cache = k_cache.data_ptr(), r.k_stride_page = k_cache.stride(0), r.k_stride_slot = k_cache.stride(1), r.k_cache_stride_head = k_cache.stride(2);
  r.v_cache = v_cache.data_ptr(), r.v_stride_page = v_cache.stride(0), r.v_stride_slot = v_cache.stride(1), r.v_cache_stride_head = v_cache.stride(2);
  r.pages = k_cache.size(0), r.page_size = k_cache.size(1);
  r.slots = slots.data_ptr<int64_t>(), r.positions = positions.data_ptr<int64_t>();
  r.cos_sin = cos_sin.data_ptr<float>(), r.cos_sin_stride = cos_sin.stride(0);
  r.max_positions = cos_sin.size(0), r.rotary = cos_sin.size(1);
  r.interleaved = interleaved ? 1 : 0;
  r.flags = VECOPS_B200_MATMUL_FLAG_ASYNC;
  r.stream = current_stream(q);
  r.device_index = static_cast<int32_t>(q.get_device());
  ErrorText error;
  error.check(vecops_b200_cache_append(&r, &error.record), "cache_append");
  return q_out;
}

// q [T,Hq,D] against the shared prefix and each sequence's own suffix in k_cache, v_cache [pages,page_size,Hkv,D]
at::Tensor sdpa_shared_prefix(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache, const at::Tensor& prefix_pages, int64_t prefix_len,
                              const at::Tensor& page_table, const at::Tensor& lengths, double scale, const c10::optional<at::Tensor>& query_starts) {
  constexpr const char* op = "sdpa_shared_prefix";
  check_operand(q, q, 3, q.scalar_type(), op, "q");
  check_operand(k_cache, q, 4, q.scalar_type(), op, "k_cache");
  check_operand(v_cache, q, 4, q.scalar_type(), op, "v_cache");
  check_operand(prefix_pages, q, 1, at::kInt, op, "prefix_pages");
  check_operand(page_table, q, 2, at::kInt, op, "page_table");
  check_operand(lengths, q, 1, at::kInt, op, "lengths");
  const int64_t t = q.size(0), hq = q.size(1), d = q.size(2), hkv = k_cache.size(2), batch = page_table.size(0);
  TORCH_CHECK(k_cache.size(3) == d && v_cache.sizes() == k_cache.sizes(), "vecops_b200.sdpa_shared_prefix: k_cache and v_cache are [pages,page_size,Hkv,", d, "]");
  TORCH_CHECK(hkv > 0 && hq % hkv == 0, "vecops_b200.sdpa_shared_prefix: ", hq, " query heads over ", hkv, " key heads");
  TORCH_CHECK(prefix_len >= 0 && k_cache.size(1) > 0 && (prefix_len + k_cache.size(1) - 1) / k_cache.size(1) <= prefix_pages.size(0),
              "vecops_b200.sdpa_shared_prefix: prefix_pages is too short for ", prefix_len, " keys in pages of ", k_cache.size(1));
  TORCH_CHECK(lengths.size(0) == batch, "vecops_b200.sdpa_shared_prefix: lengths is [", batch, "]");
  TORCH_CHECK(prefix_pages.is_contiguous() && lengths.is_contiguous(), "vecops_b200.sdpa_shared_prefix: prefix_pages and lengths must be contiguous");
  const bool ragged = query_starts.has_value() && query_starts->defined();
  if (ragged) {
    check_operand(*query_starts, q, 1, at::kInt, op, "query_starts");
    TORCH_CHECK(query_starts->size(0) == batch + 1 && query_starts->is_contiguous(), "vecops_b200.sdpa_shared_prefix: query_starts is a contiguous [", batch + 1, "]");
  } else {
    TORCH_CHECK(t == batch, "vecops_b200.sdpa_shared_prefix: without query_starts every sequence has one token (", t, " tokens, ", batch, " sequences)");
  }
  check_rows(q, op, "q");
  check_rows(k_cache, op, "k_cache");
  check_rows(v_cache, op, "v_cache");
  check_rows(page_table, op, "page_table");
  const c10::cuda::CUDAGuard guard(q.device());
  at::Tensor out = at::empty(q.sizes(), q.options());
  VecopsB200PrefixAttention r{};
  r.struct_size = sizeof(r);
  r.dtype = dtype_code(q.scalar_type());
  r.tokens = t, r.batch = batch, r.q_heads = hq, r.kv_heads = hkv, r.head_dim = d;
  r.q = q.data_ptr(), r.q_stride_token = q.stride(0), r.q_stride_head = q.stride(1);
  r.out = out.data_ptr(), r.out_stride_token = out.stride(0), r.out_stride_head = out.stride(1);
  r.k_cache = k_cache.data_ptr(), r.k_stride_page = k_cache.stride(0), r.k_stride_slot = k_cache.stride(1), r.k_stride_head = k_cache.stride(2);
  r.v_cache = v_cache.data_ptr(), r.v_stride_page = v_cache.stride(0), r.v_stride_slot = v_cache.stride(1), r.v_stride_head = v_cache.stride(2);
  r.pages = k_cache.size(0), r.page_size = k_cache.size(1);
  r.prefix_pages = prefix_pages.data_ptr<int32_t>(), r.prefix_len = prefix_len;
  r.page_table = page_table.data_ptr<int32_t>(), r.table_stride = page_table.stride(0), r.table_width = page_table.size(1);
  r.lengths = lengths.data_ptr<int32_t>();
  r.query_starts = ragged ? query_starts->data_ptr<int32_t>() : nullptr;
  r.scale = static_cast<float>(scale);
  r.flags = VECOPS_B200_MATMUL_FLAG_ASYNC;
  r.stream = current_stream(q);
  r.device_index = static_cast<int32_t>(q.get_device());
  ErrorText error;
  uint64_t need = 0;
  error.check(vecops_b200_prefix_sdpa_workspace(&r, &need, &error.record), "sdpa_shared_prefix workspace query");
  at::Tensor scratch;
  if (need != 0) {  // (torch's allocator hands out blocks on 512-byte boundaries)
    scratch = at::empty({static_cast<int64_t>(need)}, q.options().dtype(at::kByte));
    r.workspace = scratch.data_ptr();
    r.workspace_size = need;
  }
  error.check(vecops_b200_prefix_sdpa_run(&r, &error.record), "sdpa_shared_prefix");
  return out;
}

}  // namespace

TORCH_LIBRARY(vecops_b200, m) {
  m.def("matmul(Tensor a, Tensor b_nk, Tensor? column_scale=None, Tensor? cin=None, float alpha=1.0, int activation=0, float clamp_lo=0.0, "
        "float clamp_hi=0.0, ScalarType? out_dtype=None, Tensor? row_scale=None) -> Tensor");
  m.def("matmul_out(Tensor a, Tensor b_nk, Tensor(a!) c, Tensor? column_scale=None, Tensor? cin=None, float alpha=1.0, int activation=0, "
        "float clamp_lo=0.0, float clamp_hi=0.0, Tensor? row_scale=None) -> ()");
  m.def("sdpa(Tensor q, Tensor k, Tensor v, float scale, int causal=0, Tensor? key_mask=None, Tensor? bias=None, ScalarType? out_dtype=None) -> Tensor");
  m.def("quantize_blocks(Tensor x, int block_rows=1) -> (Tensor, Tensor)");
  m.def("matmul_f8_blocks(Tensor a, Tensor a_scale, Tensor b_nk, Tensor b_scale, ScalarType? out_dtype=None) -> Tensor");
  m.def("cache_append(Tensor q, Tensor k, Tensor v, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor slots, Tensor positions, Tensor cos_sin, "
        "bool interleaved=False) -> Tensor");
  m.def("sdpa_shared_prefix(Tensor q, Tensor k_cache, Tensor v_cache, Tensor prefix_pages, int prefix_len, Tensor page_table, Tensor lengths, "
        "float scale, Tensor? query_starts=None) -> Tensor");
}

TORCH_LIBRARY_IMPL(vecops_b200, CUDA, m) {
  m.impl("matmul", &matmul);
  m.impl("matmul_out", &matmul_out);
  m.impl("sdpa", &sdpa);
  m.impl("quantize_blocks", &quantize_blocks);
  m.impl("matmul_f8_blocks", &matmul_f8_blocks);
  m.impl("cache_append", &cache_append);
  m.impl("sdpa_shared_prefix", &sdpa_shared_prefix);
}
