// Torch-facing wrappers of the 8-bit block operators (blocks8.h): argument checks, outputs, tensor maps, launches on the
// current stream, autograd nodes. Registered in the extension module by ops.cpp.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cudaTypedefs.h>
#include <torch/extension.h>

#include <algorithm>
#include <atomic>

#include "blocks8.h"
#include "torch_util.h"

namespace tgo {

PFN_cuTensorMapEncodeTiled_v12000 tmap_encoder();  // ops.cpp
int num_sms();                                     // gemm.cu

namespace {

const char* const kWhat = "8-bit block operators";

int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to; }

// A packed matrix: codes [rows, 128 ceil(cols / 128)] e4m3, scale bytes (blocks8.h); the memory belongs to someone else
struct Packed {
  uint8_t* codes = nullptr;
  uint8_t* scales = nullptr;
  int64_t rows = 0, cols = 0;
  int64_t blocks() const { return up(cols, 128); }
  int64_t code_bytes() const { return rows * blocks() * 128; }
  int64_t scale_bytes() const { return up(rows, 128) * up(blocks(), 4) * 512; }
};
// Packed matrices in one allocation (a small step makes a dozen of them). The plan of a forward's checkpoint is made again
// by its backward, on the same memory.
struct Arena {
  Packed* parts[8];
  int n = 0;
  void add(Packed* p, int64_t rows, int64_t cols) {
    p->rows = rows;
    p->cols = cols;
    parts[n++] = p;
  }
  int64_t bytes() const {
    int64_t b = 0;
    for (int i = 0; i < n; ++i) b += up(parts[i]->code_bytes(), 512) * 512 + parts[i]->scale_bytes();
    return b;
  }
  at::Tensor on(const at::Tensor& as) {
    at::Tensor mem = fresh({bytes()}, at::kByte, as);
    at(mem);
    return mem;
  }
  void at(const at::Tensor& mem) {
    TORCH_CHECK(mem.is_cuda() && mem.scalar_type() == at::kByte && mem.is_contiguous() && mem.numel() == bytes() &&
                    reinterpret_cast<uintptr_t>(mem.data_ptr()) % 16 == 0, kWhat, ": the saved checkpoint has changed");
    uint8_t* p = mem.data_ptr<uint8_t>();
    for (int i = 0; i < n; ++i) {
      parts[i]->codes = p;
      p += up(parts[i]->code_bytes(), 512) * 512;
      parts[i]->scales = p;
      p += parts[i]->scale_bytes();
    }
  }
};
// as tensors of their own (what quantize_blocks returns)
Packed fresh_packed(int64_t rows, int64_t cols, const at::Tensor& as, std::vector<at::Tensor>* out) {
  Packed p;
  p.rows = rows;
  p.cols = cols;
  out->push_back(fresh({rows, p.blocks() * 128}, at::kFloat8_e4m3fn, as));
  p.codes = static_cast<uint8_t*>(out->back().data_ptr());
  out->push_back(fresh({up(rows, 128), up(p.blocks(), 4), 32, 4, 4}, at::kByte, as));
  p.scales = out->back().data_ptr<uint8_t>();
  return p;
}
Packed given_packed(const at::Tensor& codes, const at::Tensor& scales, int64_t cols, const char* what) {
  Packed p;
  p.cols = cols;
  TORCH_CHECK(codes.is_cuda() && codes.scalar_type() == at::kFloat8_e4m3fn && codes.dim() == 2 && codes.is_contiguous() &&
                  cols >= 0 && cols < (1ll << 31) - 128 && codes.size(1) == p.blocks() * 128,
              what, ": codes e4m3 [rows, 128 ceil(", cols, " / 128)], contiguous, expected");
  p.rows = codes.size(0);
  same_device(scales, codes, what);
  TORCH_CHECK(scales.scalar_type() == at::kByte && scales.is_contiguous() && p.rows < (1ll << 31) - 128 &&
                  scales.sizes() == at::IntArrayRef({up(p.rows, 128), up(p.blocks(), 4), 32, 4, 4}),
              what, ": scales uint8 [", up(p.rows, 128), ", ", up(p.blocks(), 4), ", 32, 4, 4], contiguous, expected");
  p.codes = static_cast<uint8_t*>(codes.data_ptr());
  p.scales = scales.data_ptr<uint8_t>();
  TORCH_CHECK(reinterpret_cast<uintptr_t>(p.codes) % 16 == 0 && reinterpret_cast<uintptr_t>(p.scales) % 16 == 0, what,
              ": 16-byte aligned codes and scales");
  return p;
}

// [M, K] with a row's elements side by side and rows that do not overlap; other layouts are copied
at::Tensor rows_of(const at::Tensor& t) {
  return whole_rows(t) && (t.size(0) <= 1 || t.stride(0) >= t.size(1)) ? t : t.contiguous();
}
int64_t row_stride(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }
void check_matrix(const at::Tensor& t, const char* what) {
  TORCH_CHECK(t.is_cuda() && t.dim() == 2, what, ": a CUDA matrix expected");
  TORCH_CHECK(t.size(1) >= 1 && t.size(1) < (1ll << 31) - 128 && t.size(0) < (1ll << 31) - 128, what,
              ": at least one column and fewer than 2^31 - 128 rows and columns");
}

// Packs x [M, K] (rows_of) into r (blocks along the rows) and / or c (along the columns, as the rows of x^T); sums [K] fp32:
// the column sums (with c).
struct PackJob {
  const at::Tensor& x;
  const Packed* r;
  const Packed* c;
};
Pack8Params pack_params(const PackJob& j) {
  Pack8Params p{};
  p.x = j.x.data_ptr();
  p.ld = row_stride(j.x);
  p.M = (int)j.x.size(0);
  p.K = (int)j.x.size(1);
  p.elem = elem_of(j.x, kWhat);
  if (j.r != nullptr) p.codes = j.r->codes, p.scales = j.r->scales;
  if (j.c != nullptr) p.codes_t = j.c->codes, p.scales_t = j.c->scales;
  return p;
}
void pack(const PackJob& j, float* sums = nullptr, bool add = false) {
  const int64_t M = j.x.size(0), K = j.x.size(1);
  const cudaStream_t s = at::cuda::getCurrentCUDAStream();
  if (M == 0) {
    if (sums != nullptr && !add) TORCH_CHECK(cudaMemsetAsync(sums, 0, K * sizeof(float), s) == cudaSuccess, kWhat);
    return;
  }
  Pack8Params p = pack_params(j);
  at::Tensor part;
  if (sums != nullptr) {
    part = fresh({up(M, 128), K}, at::kFloat, j.x);
    p.sums = part.data_ptr<float>();
  }
  BLOCK_LAUNCH(pack8_launch(p, s), 1);
  if (sums != nullptr) BLOCK_LAUNCH(colsum_launch(p.sums, (int)up(M, 128), (int)K, sums, add, s), 1);
}
// Several tensors (rows always wanted): one launch where they are small. Two launches cost the host some 4 us more than one,
// and their kernels' tails; past a few tiles per SM the kernels made for one type are faster.
void pack_all(std::initializer_list<PackJob> jobs) {
  Pack8Jobs all{};
  int64_t tiles = 0;
  for (const PackJob& j : jobs) tiles += up(j.x.size(0), 128) * up(j.x.size(1), 128);
  if (tiles > 4 * num_sms()) {
    for (const PackJob& j : jobs) pack(j);
    return;
  }
  for (const PackJob& j : jobs)
    if (j.x.size(0) > 0) all.job[all.n++] = pack_params(j);
  if (all.n > 0) BLOCK_LAUNCH(pack8_jobs_launch(all, at::cuda::getCurrentCUDAStream()), 1);
}

CUtensorMap codes_map(const Packed& a, uint32_t box_rows) {
  CUtensorMap m;
  const uint64_t width = a.blocks() * 128;
  cuuint64_t dims[3] = {width, (cuuint64_t)a.rows, 1};
  cuuint64_t strides[2] = {width, width * (cuuint64_t)a.rows};
  cuuint32_t box[3] = {128, box_rows, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = tmap_encoder()(&m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, a.codes, dims, strides, box, estr,
                                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TORCH_CHECK(r == CUDA_SUCCESS, "tensor map of 8-bit codes: code ", (int)r);
  return m;
}
// C [M, N] with rows ldc apart; false where a map cannot address it (the kernel then stores rows itself): base and rows off
// 16 bytes, or rows that end inside 16 bytes, which a store fills up past the row's end
bool out_map(CUtensorMap* m, const at::Tensor& C, int64_t ldc) {
  const uint64_t es = C.element_size();
  if (reinterpret_cast<uintptr_t>(C.data_ptr()) % 16 != 0 || (ldc * es) % 16 != 0 ||
      (C.size(1) * es) % 16 != 0) return false;
  const bool f32 = C.scalar_type() == at::kFloat;
  cuuint64_t dims[3] = {(cuuint64_t)C.size(1), (cuuint64_t)C.size(0), 1};
  cuuint64_t strides[2] = {ldc * es, ldc * es * (cuuint64_t)C.size(0)};
  cuuint32_t box[3] = {32, 32, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  const auto type = f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                        : C.scalar_type() == at::kHalf ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  return tmap_encoder()(m, type, 3, C.data_ptr(), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        f32 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

CUtensorMap scales_map(const Packed& a, uint32_t box_tiles) {
  CUtensorMap m;
  const uint64_t quads = up(a.blocks(), 4);
  cuuint64_t dims[3] = {128, quads, (cuuint64_t)up(a.rows, 128)};
  cuuint64_t strides[2] = {512, quads * 512};
  cuuint32_t box[3] = {128, 1, box_tiles};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = tmap_encoder()(&m, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, a.scales, dims, strides, box, estr,
                                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TORCH_CHECK(r == CUDA_SUCCESS, "tensor map of 8-bit scales: code ", (int)r);
  return m;
}

// a product C [M, N] (+)= a b^T (+ bias)
struct Product {
  const Packed &a, &b;
  const at::Tensor& C;
  const float* bias;
  bool add;
};
std::atomic<int> g_tile{-1};  // for comparisons of the variants: -1 chooses
// The tile whose products end first on the whole GPU, by the cycles of a tile (gemm8.cu). Measured at 32768 x 6144 x 2048: 436
// us for 128 x 128, 287 for 256 x 192, 305 for 256 x 256; x 2048 x 6144: 418, 281 and 264; 2047 x 777 x 1000: 17, 21 and 26.
Gemm8Tile tile_of(const Gemm8Params& p) {
  if (g_tile >= 0) return (Gemm8Tile)g_tile.load();
  const int rows[3] = {128, 256, 256}, cols[3] = {128, 192, 256};
  Gemm8Tile best = TILE_128x128;
  int64_t least = 0;
  for (int k = 0; k < 3; ++k) {
    const int64_t units = k == 0 ? num_sms() : num_sms() / 2;
    int64_t tiles[2] = {0, 0}, cost[2] = {0, 0}, all = 0, work = 0;
    for (int i = 0; i < p.n; ++i) all += tiles[i] = up(p.q[i].M, rows[k]) * up(p.q[i].N, cols[k]);
    for (int i = 0; i < p.n; ++i) work += tiles[i] * (cost[i] = gemm8_tile_cycles(p.q[i], (Gemm8Tile)k, all > units));
    // one product: whole waves; two: the first one's waves, or all work and half of a second one's tile
    const int64_t ends = std::max(up(tiles[0], units) * cost[0], p.n == 1 ? 0 : work / units + cost[1] / 2);
    if (k == 0 || ends < least) {
      least = ends;
      best = (Gemm8Tile)k;
    }
  }
  return best;
}

// One or two products in a launch
void products(std::initializer_list<Product> list, int* err) {
  Gemm8Params p{};
  Gemm8Maps t;
  const Product* of[2] = {nullptr, nullptr};
  for (const Product& w : list) {
    TORCH_CHECK(w.a.cols == w.b.cols, "gemm_blocks: sums over ", w.a.cols, " and ", w.b.cols);
    if (w.a.rows == 0 || w.b.rows == 0) continue;
    if (w.a.cols == 0) {  // a sum of nothing
      TORCH_CHECK(w.bias == nullptr, "gemm_blocks: a bias of a sum of nothing");
      if (!w.add) w.C.zero_();
      continue;
    }
    of[p.n++] = &w;
  }
  if (p.n == 2 && of[0]->a.cols < of[1]->a.cols) std::swap(of[0], of[1]);  // the longer sums first
  for (int i = 0; i < p.n; ++i) {
    const Product& w = *of[i];
    Gemm8Problem& q = p.q[i];
    q.M = (int)w.a.rows;
    q.N = (int)w.b.rows;
    q.kb = (int)w.a.blocks();
    q.sfa = w.a.scales;
    q.sfb = w.b.scales;
    q.C = w.C.data_ptr();
    q.ldc = row_stride(w.C);
    q.bias = w.bias;
    q.add = w.add;
    q.elem = elem_of(w.C, "gemm_blocks");
    // The tensor core's fp32 sums drop what does not fit their 24 bits instead of rounding: a sum of one sign over 32768
    // lost 3.6e-5 of itself, 1.3e-6 over 4096. Sums that are returned in fp32 are joined from parts of 4096.
    q.chunk_kb = q.elem == ELEM_F32 ? 32 : (int)up(q.kb, 4) * 4;
    q.c_tma = out_map(&t.c[i], w.C, q.ldc);
  }
  if (p.n == 0) return;
  p.err = err;
  const Gemm8Tile tile = tile_of(p);
  for (int i = 0; i < p.n; ++i) {
    t.a[i] = codes_map(of[i]->a, 128);
    t.b[i] = codes_map(of[i]->b, tile == TILE_PAIR_192 ? 96 : 128);
    if (tile != TILE_128x128) {
      t.sa[i] = scales_map(of[i]->a, 1);
      t.sb[i] = scales_map(of[i]->b, 2);
    }
    if (!p.q[i].c_tma) t.c[i] = t.a[i];
  }
  BLOCK_LAUNCH(gemm8_launch(t, p, tile, at::cuda::getCurrentCUDAStream()), 1);
}
void product(const Packed& a, const Packed& b, const at::Tensor& C, const float* bias, bool add, int* err) {
  products({{a, b, C, bias, add}}, err);
}

void small_vector(const OptT& bias, int64_t n, const at::Tensor& as, const char* what) {
  if (!given(bias)) return;
  same_device(*bias, as, what);
  TORCH_CHECK(bias->is_floating_point() && bias->dim() == 1 && bias->size(0) == n, what, ": bias [", n, "] expected");
}
// the bias in fp32 (a copy where it is not)
at::Tensor bias_f32(const OptT& bias) {
  if (!given(bias)) return at::Tensor();
  if (bias->scalar_type() == at::kFloat && bias->is_contiguous()) return *bias;
  return bias->detach().to(at::kFloat).contiguous();
}
const float* ptr_f32(const at::Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }

// ------------------------------------------------------------------------------------------------ packing, products
std::vector<at::Tensor> pack8(at::Tensor x, bool rows, bool cols) {
  TORCH_CHECK(rows || cols, "quantize_blocks: a side");
  check_matrix(x, "quantize_blocks");
  const c10::cuda::CUDAGuard guard(x.device());
  x = rows_of(x.detach());
  elem_of(x, "quantize_blocks");
  std::vector<at::Tensor> out;
  Packed r, c;
  if (rows) r = fresh_packed(x.size(0), x.size(1), x, &out);
  if (cols) c = fresh_packed(x.size(1), x.size(0), x, &out);
  pack({x, rows ? &r : nullptr, cols ? &c : nullptr});
  return out;
}

at::Tensor unpack8(at::Tensor codes, at::Tensor scales, int64_t cols, at::ScalarType type) {
  const Packed p = given_packed(codes, scales, cols, "dequantize_blocks");
  const c10::cuda::CUDAGuard guard(codes.device());
  at::Tensor out = fresh({p.rows, cols}, type, codes);
  const int elem = elem_of(out, "dequantize_blocks");
  if (out.numel() > 0)
    BLOCK_LAUNCH(unpack8_launch(p.codes, p.scales, (int)p.rows, (int)cols, out.data_ptr(), cols, elem,
                                at::cuda::getCurrentCUDAStream()), 1);
  return out;
}

at::Tensor gemm8(at::Tensor a, at::Tensor as, at::Tensor b, at::Tensor bs, int64_t cols, at::ScalarType type, OptT out,
                 OptT bias, bool add, at::Tensor err) {
  const Packed p = given_packed(a, as, cols, "gemm_blocks: a"), q = given_packed(b, bs, cols, "gemm_blocks: b");
  same_device(b, a, "gemm_blocks: b");
  const c10::cuda::CUDAGuard guard(a.device());
  small_vector(bias, q.rows, a, "gemm_blocks");
  at::Tensor C = given(out) ? *out : fresh({p.rows, q.rows}, type, a);
  same_device(C, a, "gemm_blocks: out");
  TORCH_CHECK(C.dim() == 2 && C.size(0) == p.rows && C.size(1) == q.rows && whole_rows(C) &&
                  (C.size(0) <= 1 || C.stride(0) >= C.size(1)), "gemm_blocks: out [", p.rows, ", ", q.rows,
              "] with contiguous rows expected");
  TORCH_CHECK(!(C.requires_grad() && at::GradMode::is_enabled()), "gemm_blocks: out must not require a gradient");
  TORCH_CHECK(!add || (given(out) && C.scalar_type() == at::kFloat && !given(bias)),
              "gemm_blocks: adding takes an fp32 out and no bias");
  const at::Tensor b32 = bias_f32(bias);
  product(p, q, C, ptr_f32(b32), add, err_word(err, a));
  return C;
}

// ----------------------------------------------------------------------------------------------------------- linear
// y = Q(x) w^T + bias; few rows of x in one launch, packed on the way
void times_held(const at::Tensor& x, const Packed& w, const at::Tensor& y, const float* bias, int* err) {
  if (y.numel() == 0) return;
  if (x.size(0) <= kFewRows) {
    FewRowsParams p{};
    p.x = x.data_ptr();
    p.ldx = row_stride(x);
    p.codes = w.codes;
    p.scales = w.scales;
    p.bias = bias;
    p.y = y.data_ptr();
    p.M = (int)x.size(0);
    p.N = (int)w.rows;
    p.K = (int)w.cols;
    BLOCK_LAUNCH(few_rows_launch(p, elem_of(x, kWhat), at::cuda::getCurrentCUDAStream()), 1);
    return;
  }
  Packed q;
  Arena arena;
  arena.add(&q, x.size(0), x.size(1));
  const at::Tensor mem = arena.on(x);
  pack({x, &q, nullptr});
  product(q, w, y, bias, false, err);
}
void no_graph(std::initializer_list<const at::Tensor*> ts, const char* what) {
  TORCH_CHECK(!wants_grad(ts, kWhat), what, ": a weight held in 8 bits passes no gradient on (use torch.no_grad() or detach x)");
}
// Q(x) W^T + bias with W held in 8 bits; no gradient
at::Tensor linear8_frozen(at::Tensor x, at::Tensor codes, at::Tensor scales, int64_t cols, OptT bias, at::Tensor err) {
  const Packed w = given_packed(codes, scales, cols, "linear_blocks: weight");
  same_device(codes, x, "linear_blocks: weight");
  check_matrix(x, "linear_blocks");
  elem_of(x, "linear_blocks");
  TORCH_CHECK(x.size(1) == cols && w.rows >= 1, "linear_blocks: x [..., ", cols, "] expected, got ", x.size(1), " columns");
  const at::Tensor b = or_undefined(bias);
  no_graph({&x, &b}, "linear_blocks");
  const c10::cuda::CUDAGuard guard(x.device());
  small_vector(bias, w.rows, x, "linear_blocks");
  x = rows_of(x);
  const at::Tensor b32 = bias_f32(bias);
  at::Tensor y = fresh({x.size(0), w.rows}, x.scalar_type(), x);
  times_held(x, w, y, ptr_f32(b32), err_word(err, x));
  return y;
}

// The operands of a backward product are packed along the axis that it sums over: x^T and W^T are written while the
// forward packs x and W. x itself is not kept: its checkpoint is the operand of the weight's gradient.
// In one launch: a layer's input gradient dx = r wt^T (null: not wanted) and its weight's gradient dw = c xt^T where autograd
// or the leaf wants it
void gradients(const at::Tensor* dx, const Packed& r, const Packed& wt, const WeightGrad& dw, const Packed& c, const Packed& xt,
               int* err) {
  if (dx != nullptr && dw.g.defined()) products({{r, wt, *dx, nullptr, false}, {c, xt, dw.g, nullptr, dw.add}}, err);
  else if (dx != nullptr) product(r, wt, *dx, nullptr, false, err);
  else if (dw.g.defined()) product(c, xt, dw.g, nullptr, dw.add, err);
}
void notify(std::initializer_list<const WeightGrad*> gs) {
  if (!grad_ready().on) return;
  py::gil_scoped_acquire gil;
  for (const WeightGrad* g : gs)
    if (g->direct) grad_ready().notify(g->w);
}

struct Linear8Fn : public torch::autograd::Function<Linear8Fn> {
  static at::Tensor forward(AutogradContext* ctx, at::Tensor x, at::Tensor w, OptT bias, at::Tensor err) {
    at::AutoDispatchBelowADInplaceOrView below;
    const bool dx = x.requires_grad(), dw = w.requires_grad();
    const int64_t M = x.size(0), K = x.size(1), N = w.size(0);
    Packed xr, xt, wr, wt;
    Arena now, later;
    now.add(&xr, M, K);
    now.add(&wr, N, K);
    if (dw) later.add(&xt, K, M);
    if (dx) later.add(&wt, K, N);
    const at::Tensor mem = now.on(x), checkpoint = later.on(x);
    pack_all({{x, &xr, dw ? &xt : nullptr}, {w, &wr, dx ? &wt : nullptr}});
    at::Tensor y = fresh({M, N}, x.scalar_type(), x);
    const at::Tensor b32 = bias_f32(bias);
    product(xr, wr, y, ptr_f32(b32), false, err_word(err, x));
    ctx->save_for_backward({checkpoint});
    // a weight or bias that is no part of the graph now gets no gradient, whatever its flag is when the backward runs
    if (dw) ctx->saved_data["w"] = w;
    if (given(bias) && bias->requires_grad()) ctx->saved_data["bias"] = *bias;
    ctx->saved_data["K"] = K;
    ctx->saved_data["err"] = err;
    ctx->saved_data["of"] = (dx ? 1 : 0) + (dw ? 2 : 0);
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    first_order_only(kWhat);
    const auto saved = ctx->get_saved_variables();
    const at::Tensor dy = rows_of(grads[0]);
    const c10::cuda::CUDAGuard guard(dy.device());
    const int64_t M = dy.size(0), N = dy.size(1), of = ctx->saved_data["of"].toInt();
    const bool dx = of & 1;
    const at::Tensor err = ctx->saved_data["err"].toTensor();
    int* const e = err_word(err, dy);
    const WeightGrad gw(ctx, "w"), gb(ctx, "bias");
    const int64_t K = ctx->saved_data["K"].toInt();
    Packed xt, wt, r, c;
    Arena before, now;
    if (of & 2) before.add(&xt, K, M);
    if (of & 1) before.add(&wt, K, N);
    before.at(saved[0]);
    // the bias' sums are fp32 wherever they go
    at::Tensor sums = gb.g.defined() ? (gb.g.scalar_type() == at::kFloat ? gb.g : fresh({N}, at::kFloat, dy)) : at::Tensor();
    const bool dw = gw.g.defined(), cols = dw || sums.defined();
    if (dx) now.add(&r, M, N);
    if (cols) now.add(&c, N, M);
    const at::Tensor mem = now.on(dy);
    if (dx || cols) pack({dy, dx ? &r : nullptr, cols ? &c : nullptr}, sums.defined() ? sums.data_ptr<float>() : nullptr, gb.add);
    variable_list out(4);
    if (dx) out[0] = fresh({M, K}, dy.scalar_type(), dy);
    gradients(dx ? &out[0] : nullptr, r, wt, gw, c, xt, e);
    out[1] = gw.put();
    if (sums.defined()) {
      if (gb.g.scalar_type() != at::kFloat) gb.g.copy_(sums);
      out[2] = gb.put();
    }
    notify({&gw, &gb});
    return out;
  }
};

at::Tensor linear8(at::Tensor x, at::Tensor w, OptT bias, at::Tensor err) {
  check_matrix(x, "linear_blocks");
  check_matrix(w, "linear_blocks: weight");
  same_device(w, x, "linear_blocks: weight");
  TORCH_CHECK(x.size(1) == w.size(1) && w.size(0) >= 1, "linear_blocks: x [..., K] and weight [N, K] expected, got ",
              x.sizes(), " and ", w.sizes());
  elem_of(x, "linear_blocks");
  elem_of(w, "linear_blocks: weight");
  const c10::cuda::CUDAGuard guard(x.device());
  small_vector(bias, w.size(0), x, "linear_blocks");
  x = rows_of(x);
  const at::Tensor b = or_undefined(bias);
  if (wants_grad({&x, &w, &b}, kWhat)) {
    if (!whole_rows(w)) w = w.contiguous();
    return Linear8Fn::apply(x, w, bias, err);
  }
  w = rows_of(w);
  Packed xr, wr;
  Arena now;
  now.add(&xr, x.size(0), x.size(1));
  now.add(&wr, w.size(0), w.size(1));
  const at::Tensor mem = now.on(x);
  pack_all({{x, &xr, nullptr}, {w, &wr, nullptr}});
  at::Tensor y = fresh({x.size(0), w.size(0)}, x.scalar_type(), x);
  const at::Tensor b32 = bias_f32(bias);
  product(xr, wr, y, ptr_f32(b32), false, err_word(err, x));
  return y;
}

// ----------------------------------------------------------------------------------------------------------- SwiGLU
// plain {cols, rows, 1} map with a {side, side, 1} box
CUtensorMap tile_map(const void* base, CUtensorMapDataType type, uint64_t size, uint64_t cols, uint64_t rows, uint64_t ld,
                     uint32_t side = 128) {
  CUtensorMap m;
  cuuint64_t dims[3] = {cols, rows, 1};
  cuuint64_t strides[2] = {ld * size, ld * size * rows};
  cuuint32_t box[3] = {side, side, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = tmap_encoder()(&m, type, 3, const_cast<void*>(base), dims, strides, box, estr,
                                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TORCH_CHECK(r == CUDA_SUCCESS, "tensor map of activations: code ", (int)r);
  return m;
}
CUtensorMap tile_map(const at::Tensor& t) {
  const auto type = t.scalar_type() == at::kFloat  ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                    : t.scalar_type() == at::kHalf ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  return tile_map(t.data_ptr(), type, t.element_size(), t.size(1), t.size(0), t.size(1));
}
void swiglu_forward(const at::Tensor& ab, at::Tensor* g, const Packed* ck, const Packed* g8, const Packed* g8t, int* err) {
  const int64_t M = ab.size(0), H = ab.size(1) / 2;
  if (g != nullptr) *g = fresh({M, H}, ab.scalar_type(), ab);
  if (M == 0) return;
  Swiglu8Params p{};
  p.ab = ab.data_ptr();
  p.ld = row_stride(ab);
  p.M = (int)M;
  p.H = (int)H;
  if (g != nullptr) p.g = g->data_ptr();
  if (ck != nullptr) p.ck = ck->codes, p.ck_scales = ck->scales;
  if (g8 != nullptr) p.g8 = g8->codes, p.g8_scales = g8->scales;
  if (g8t != nullptr) p.g8t = g8t->codes, p.g8t_scales = g8t->scales;
  CUtensorMap map;
  if (g8 != nullptr) {  // ab is the contiguous output of a product
    map = tile_map(ab);
    p.map = &map;
    p.err = err;
  }
  BLOCK_LAUNCH(swiglu8_fwd_launch(p, elem_of(ab, "swiglu_blocks"), at::cuda::getCurrentCUDAStream()), 1);
}
void swiglu_backward(const at::Tensor& dg, const Packed& ck, int64_t H, at::Tensor* dab, const Packed* d8, const Packed* d8t,
                     int* err) {
  const int64_t M = dg.size(0);
  if (dab != nullptr) *dab = fresh({M, 2 * H}, dg.scalar_type(), dg);
  if (M == 0) return;
  Swiglu8BwdParams p{};
  p.dg = dg.data_ptr();
  p.ld = row_stride(dg);
  p.ck = ck.codes;
  p.ck_scales = ck.scales;
  p.M = (int)M;
  p.H = (int)H;
  if (dab != nullptr) p.dab = dab->data_ptr();
  if (d8 != nullptr) p.d8 = d8->codes, p.d8_scales = d8->scales;
  if (d8t != nullptr) p.d8t = d8t->codes, p.d8t_scales = d8t->scales;
  CUtensorMap map, ck_map;
  if (d8 != nullptr) {  // dg is the contiguous output of a product
    map = tile_map(dg);
    ck_map = tile_map(p.ck, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, 2 * H, M, 2 * H);
    p.map = &map;
    p.ck_map = &ck_map;
    p.err = err;
  }
  BLOCK_LAUNCH(swiglu8_bwd_launch(p, elem_of(dg, "swiglu_blocks"), at::cuda::getCurrentCUDAStream()), 1);
}

// [a | b] = x w^T rounded to `like`'s type, g = silu(a) b: the checkpoint (ck, or null), g along its rows and (g8t, or null) its
// columns. 16-bit types: one launch, the activations stay on the chip; fp32 (whose values do not fit the registers): two.
void product_swiglu(const Packed& x, const Packed& w, const at::Tensor& like, const Packed* ck, const Packed& g8,
                    const Packed* g8t, int* err) {
  const int64_t M = x.rows, H = w.rows / 2;
  if (M == 0) return;
  const int elem = elem_of(like, kWhat);
  if (elem == ELEM_F32) {
    at::Tensor ab = fresh({M, 2 * H}, like.scalar_type(), like);
    product(x, w, ab, nullptr, false, err);
    swiglu_forward(ab, nullptr, ck, &g8, g8t, err);
    return;
  }
  Gemm8Params p{};
  Gemm8Problem& q = p.q[0];
  p.n = 1;
  p.err = err;
  q.M = (int)M;
  q.N = (int)(2 * H);
  q.kb = (int)x.blocks();
  q.sfa = x.scales;
  q.sfb = w.scales;
  q.elem = elem;
  q.chunk_kb = (int)up(q.kb, 4) * 4;
  Gemm8Maps t;
  t.a[0] = codes_map(x, 128);
  t.b[0] = codes_map(w, 128);
  t.sa[0] = scales_map(x, 1);
  t.sb[0] = scales_map(w, 1);
  t.c[0] = t.a[0];
  Gemm8SwigluOut o{};
  if (ck != nullptr) o.ck = ck->codes, o.ck_scales = ck->scales;
  o.g8 = g8.codes;
  o.g8_scales = g8.scales;
  CUtensorMap g8t_map;
  if (g8t != nullptr) {
    g8t_map = tile_map(g8t->codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, g8t->blocks() * 128, H, g8t->blocks() * 128, 32);
    o.g8t = g8t->codes;
    o.g8t_scales = g8t->scales;
    o.g8t_map = &g8t_map;
  }
  BLOCK_LAUNCH(gemm8_swiglu_launch(t, p, o, at::cuda::getCurrentCUDAStream()), 1);
}

struct Swiglu8Fn : public torch::autograd::Function<Swiglu8Fn> {
  static at::Tensor forward(AutogradContext* ctx, at::Tensor ab) {
    at::AutoDispatchBelowADInplaceOrView below;
    at::Tensor g;
    Packed ck;
    Arena later;
    later.add(&ck, ab.size(0), 2 * up(ab.size(1) / 2, 128) * 128);
    ctx->save_for_backward({later.on(ab)});
    swiglu_forward(ab, &g, &ck, nullptr, nullptr, nullptr);
    return g;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    first_order_only(kWhat);
    const auto saved = ctx->get_saved_variables();
    const at::Tensor dg = rows_of(grads[0]);
    const c10::cuda::CUDAGuard guard(dg.device());
    at::Tensor dab;
    Packed ck;
    Arena before;
    before.add(&ck, dg.size(0), 2 * up(dg.size(1), 128) * 128);
    before.at(saved[0]);
    swiglu_backward(dg, ck, dg.size(1), &dab, nullptr, nullptr, nullptr);
    return {dab};
  }
};
at::Tensor swiglu8(at::Tensor ab) {
  check_matrix(ab, "swiglu_blocks");
  TORCH_CHECK(ab.size(1) % 2 == 0 && ab.size(1) < (1ll << 31) - 512, "swiglu_blocks: an even number of columns");
  elem_of(ab, "swiglu_blocks");
  const c10::cuda::CUDAGuard guard(ab.device());
  ab = rows_of(ab);
  if (wants_grad({&ab}, kWhat)) return Swiglu8Fn::apply(ab);
  at::Tensor g;
  swiglu_forward(ab, &g, nullptr, nullptr, nullptr, nullptr);
  return g;
}

// -------------------------------------------------------------------------------------------------------------- MLP
// what the backward reads: x^T (of bit 2: in_proj's gradient), W1^T (bit 1: x's gradient), W2^T and [a | b] (either), g^T (bit 4:
// out_proj's gradient)
struct MlpCheckpoint {
  Packed xt, w1t, w2t, ck, gt;
  Arena arena;
  MlpCheckpoint(int64_t M, int64_t K, int64_t H, int64_t N, int64_t of) {
    if (of & 2) arena.add(&xt, K, M);
    if (of & 1) arena.add(&w1t, K, 2 * H);
    if (of & 3) arena.add(&w2t, H, N);
    if (of & 3) arena.add(&ck, M, 2 * H);
    if (of & 4) arena.add(&gt, H, M);
  }
};
struct Mlp8Fn : public torch::autograd::Function<Mlp8Fn> {
  static at::Tensor forward(AutogradContext* ctx, at::Tensor x, at::Tensor w1, at::Tensor w2, at::Tensor err) {
    at::AutoDispatchBelowADInplaceOrView below;
    const int64_t M = x.size(0), K = x.size(1), H = w2.size(1), N = w2.size(0);
    const int64_t of = (x.requires_grad() ? 1 : 0) + (w1.requires_grad() ? 2 : 0) + (w2.requires_grad() ? 4 : 0);
    MlpCheckpoint c(M, K, H, N, of);
    const at::Tensor checkpoint = c.arena.on(x);
    Packed xr, w1r, w2r, g8;
    Arena now;
    now.add(&xr, M, K);
    now.add(&w1r, 2 * H, K);
    now.add(&w2r, N, H);
    now.add(&g8, M, H);
    const at::Tensor mem = now.on(x);
    pack_all({{x, &xr, of & 2 ? &c.xt : nullptr}, {w1, &w1r, of & 1 ? &c.w1t : nullptr}, {w2, &w2r, of & 3 ? &c.w2t : nullptr}});
    int* const e = err_word(err, x);
    product_swiglu(xr, w1r, x, of & 3 ? &c.ck : nullptr, g8, of & 4 ? &c.gt : nullptr, e);
    at::Tensor y = fresh({M, N}, x.scalar_type(), x);
    product(g8, w2r, y, nullptr, false, e);
    ctx->save_for_backward({checkpoint});
    if (of & 2) ctx->saved_data["w1"] = w1;  // as in Linear8Fn
    if (of & 4) ctx->saved_data["w2"] = w2;
    ctx->saved_data["K"] = K;
    ctx->saved_data["H"] = H;
    ctx->saved_data["err"] = err;
    ctx->saved_data["of"] = of;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    first_order_only(kWhat);
    const auto saved = ctx->get_saved_variables();
    const at::Tensor dy = rows_of(grads[0]);
    const c10::cuda::CUDAGuard guard(dy.device());
    const int64_t of = ctx->saved_data["of"].toInt();
    const int64_t M = dy.size(0), N = dy.size(1), H = ctx->saved_data["H"].toInt(), K = ctx->saved_data["K"].toInt();
    const at::Tensor err = ctx->saved_data["err"].toTensor();
    int* const e = err_word(err, dy);
    const WeightGrad g1(ctx, "w1"), g2(ctx, "w2");
    const bool dx = of & 1, dw1 = g1.g.defined(), dw2 = g2.g.defined(), up_too = dx || dw1;
    MlpCheckpoint c(M, K, H, N, of);
    c.arena.at(saved[0]);
    Packed dyr, dyt, d8, d8t;
    Arena now;
    if (up_too) now.add(&dyr, M, N);
    if (dw2) now.add(&dyt, N, M);
    if (up_too) now.add(&d8, M, 2 * H);
    if (up_too) now.add(&d8t, 2 * H, M);
    const at::Tensor mem = now.on(dy);
    if (up_too || dw2) pack({dy, up_too ? &dyr : nullptr, dw2 ? &dyt : nullptr});
    variable_list out(4);
    at::Tensor dg;
    if (up_too) dg = fresh({M, H}, dy.scalar_type(), dy);
    gradients(up_too ? &dg : nullptr, dyr, c.w2t, g2, dyt, c.gt, e);
    out[2] = g2.put();
    if (up_too) {
      swiglu_backward(dg, c.ck, H, nullptr, &d8, &d8t, e);
      dg = at::Tensor();
      if (dx) out[0] = fresh({M, K}, dy.scalar_type(), dy);
      gradients(dx ? &out[0] : nullptr, d8, c.w1t, g1, d8t, c.xt, e);
      out[1] = g1.put();
    }
    notify({&g2, &g1});
    return out;
  }
};
at::Tensor mlp8(at::Tensor x, at::Tensor w1, at::Tensor w2, at::Tensor err) {
  check_matrix(x, "mlp_blocks");
  check_matrix(w1, "mlp_blocks: in_proj");
  check_matrix(w2, "mlp_blocks: out_proj");
  same_device(w1, x, "mlp_blocks: in_proj");
  same_device(w2, x, "mlp_blocks: out_proj");
  TORCH_CHECK(x.size(1) == w1.size(1) && w1.size(0) == 2 * w2.size(1) && w2.size(0) >= 1 && w2.size(1) % 128 == 0,
              "mlp_blocks: x [..., K], in_proj [2 H, K] and out_proj [N, H] with H a multiple of 128 expected, got ",
              x.sizes(), ", ", w1.sizes(), " and ", w2.sizes());
  elem_of(x, "mlp_blocks");
  elem_of(w1, "mlp_blocks: in_proj");
  elem_of(w2, "mlp_blocks: out_proj");
  const c10::cuda::CUDAGuard guard(x.device());
  x = rows_of(x);
  if (wants_grad({&x, &w1, &w2}, kWhat)) {
    if (!whole_rows(w1)) w1 = w1.contiguous();
    if (!whole_rows(w2)) w2 = w2.contiguous();
    return Mlp8Fn::apply(x, w1, w2, err);
  }
  w1 = rows_of(w1);
  w2 = rows_of(w2);
  Packed xr, w1r, w2r, g8;
  Arena now;
  now.add(&xr, x.size(0), x.size(1));
  now.add(&w1r, w1.size(0), w1.size(1));
  now.add(&w2r, w2.size(0), w2.size(1));
  now.add(&g8, x.size(0), w2.size(1));
  const at::Tensor mem = now.on(x);
  pack_all({{x, &xr, nullptr}, {w1, &w1r, nullptr}, {w2, &w2r, nullptr}});
  int* const e = err_word(err, x);
  at::Tensor y = fresh({x.size(0), w2.size(0)}, x.scalar_type(), x);
  product_swiglu(xr, w1r, x, nullptr, g8, nullptr, e);
  product(g8, w2r, y, nullptr, false, e);
  return y;
}

// with both weights held in 8 bits; no gradient
at::Tensor mlp8_frozen(at::Tensor x, at::Tensor c1, at::Tensor s1, at::Tensor c2, at::Tensor s2, int64_t K, int64_t H,
                       at::Tensor err) {
  const Packed w1 = given_packed(c1, s1, K, "mlp_blocks: in_proj"), w2 = given_packed(c2, s2, H, "mlp_blocks: out_proj");
  same_device(c1, x, "mlp_blocks: in_proj");
  same_device(c2, x, "mlp_blocks: out_proj");
  check_matrix(x, "mlp_blocks");
  elem_of(x, "mlp_blocks");
  TORCH_CHECK(x.size(1) == K && w1.rows == 2 * H && H >= 1 && w2.rows >= 1 && H % 128 == 0,
              "mlp_blocks: x [..., K], in_proj [2 H, K] and out_proj [N, H] with H a multiple of 128 expected");
  no_graph({&x}, "mlp_blocks");
  const c10::cuda::CUDAGuard guard(x.device());
  x = rows_of(x);
  int* const e = err_word(err, x);
  const int64_t M = x.size(0);
  at::Tensor y = fresh({M, w2.rows}, x.scalar_type(), x);
  Packed xr, g8;
  Arena now;
  if (M > kFewRows) now.add(&xr, M, K);
  now.add(&g8, M, H);
  const at::Tensor mem = now.on(x);
  if (M > kFewRows) {
    pack({x, &xr, nullptr});
    product_swiglu(xr, w1, x, nullptr, g8, nullptr, e);
  } else {
    at::Tensor ab = fresh({M, 2 * H}, x.scalar_type(), x);
    times_held(x, w1, ab, nullptr, e);
    swiglu_forward(ab, nullptr, nullptr, &g8, nullptr, e);
  }
  product(g8, w2, y, nullptr, false, e);
  return y;
}

}  // namespace

void bind_blocks8(pybind11::module_& m) {
  m.def("pack8", &pack8, "rows and / or columns of a matrix in 8-bit blocks -> codes, scales of each");
  m.def("unpack8", [](at::Tensor codes, at::Tensor scales, int64_t cols, py::object dtype) {
    return unpack8(codes, scales, cols, torch::python::detail::py_object_to_dtype(dtype));
  }, "the values that 8-bit blocks stand for");
  m.def("gemm8", [](at::Tensor a, at::Tensor as, at::Tensor b, at::Tensor bs, int64_t cols, py::object dtype, OptT out,
                    OptT bias, bool add, at::Tensor err) {
    return gemm8(a, as, b, bs, cols, torch::python::detail::py_object_to_dtype(dtype), out, bias, add, err);
  }, "C (+)= a b^T (+ bias) of packed matrices");
  m.def("set_gemm8_tile", [](int64_t t) {
    TORCH_CHECK(t >= -1 && t <= 2, "set_gemm8_tile: -1 (chosen by size), 0 (128 x 128), 1 (256 x 192), 2 (256 x 256)");
    g_tile = (int)t;
  }, "tile of the 8-bit products (A/B runs)");
  m.def("linear8_frozen", &linear8_frozen, "x times a weight held in 8 bits");
  m.def("linear8", &linear8, "linear layer on 8-bit products, forward and backward");
  m.def("swiglu8", &swiglu8, "silu(a) b with its input kept in 8 bits for the backward");
  m.def("mlp8_frozen", &mlp8_frozen, "SwiGLU MLP with weights held in 8 bits");
  m.def("mlp8", &mlp8, "SwiGLU MLP on 8-bit products, forward and backward");
}

}  // namespace tgo
