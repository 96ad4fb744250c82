// Torch bindings of the 8-bit block matrices and of layer norm.  Each function
// is one direction of an operator: it checks its arguments, allocates outputs
// and workspaces from torch's caching allocator (so they are safe in captured
// graphs) and launches on the current stream of the arguments' device.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <hip/hip_runtime_api.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <tuple>

#include "riqn_kernels.h"

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

void* stream_of(const Tensor& t) {
    return (void*)at::cuda::getCurrentCUDAStream(t.device().index()).stream();
}

void launched(int err, const char* what) {
    TORCH_CHECK(err == 0, what, ": ", hipGetErrorString((hipError_t)err));
}

int type_code(at::ScalarType t, const char* name) {
    switch (t) {
        case torch::kFloat32: return 0;
        case torch::kBFloat16: return 1;
        case torch::kFloat16: return 2;
        default:
            TORCH_CHECK(false, name, " must be float32, bfloat16 or float16, got ",
                        at::toString(t));
    }
}

// A tracer sees the allocations of a call and none of its kernels: what it
// records would return memory that nobody wrote.
void check_call() {
    TORCH_CHECK(!torch::jit::tracer::isTracing(),
                "this operator's GPU kernels cannot be traced");
}

// The kernels read and write memory.  A tensor that stands for others (a
// subclass that holds them, a transform's), for shapes alone or for zeros has
// none, and its address is null.
void check_memory(const Tensor& t) {
    using c10::DispatchKey;
    TORCH_CHECK(t.has_storage() &&
                    !t.key_set().has_any(c10::DispatchKeySet(
                        {DispatchKey::Python, DispatchKey::Functionalize,
                         DispatchKey::ZeroTensor})),
                "a tensor without memory of its own is not for this operator");
}

// torch's allocator, unless a mode hands out something else in its place
Tensor fresh(c10::IntArrayRef sizes, const at::TensorOptions& options) {
    Tensor t = torch::empty(sizes, options);
    check_memory(t);
    return t;
}

// What an operator is handed: forward-mode derivatives are not there, and a
// tangent that the kernels cannot see would count as zero.
void check_given(const Tensor& t) {
    check_memory(t);
    TORCH_CHECK(!t._fw_grad(0).defined(),
                "this operator has no forward-mode derivatives");
}
void check_given(const OptTensor& t) {
    if (t) check_given(*t);
}

// a matrix whose rows are contiguous and any stride apart
void check_rows(const Tensor& x, const char* name) {
    TORCH_CHECK(x.is_cuda(), name, " must be on GPU");
    TORCH_CHECK(x.dim() == 2, name, " must have 2 dimensions");
    TORCH_CHECK(x.size(1) <= 1 || x.stride(1) == 1 || x.numel() == 0, name,
                " must have contiguous rows");
    TORCH_CHECK(x.size(0) <= (1 << 30) && x.size(1) <= (1 << 24), name,
                " must have at most 2^30 rows and 2^24 columns");
}

void check_vector(const Tensor& v, int64_t n, const Tensor& like,
                  const char* name) {
    TORCH_CHECK(v.device() == like.device(), name, " must be on ", like.device());
    TORCH_CHECK(v.dim() == 1 && v.size(0) == n, name, " must have ", n,
                " elements in 1 dimension");
    TORCH_CHECK(v.is_contiguous() && !v.is_neg(), name,
                " must be contiguous, and no negated view");
}

int64_t blocks_of(int64_t n) { return (n + 127) / 128; }
int64_t padded4(int64_t n) { return (n + 3) / 4 * 4; }

// a matrix in 8-bit blocks where it lies; the memory is another's
struct Mat {
    uint8_t *q, *scale;
    int64_t rows, block_rows;
};

struct Blocks {
    Tensor q, scale;
    int64_t rows, block_rows;
    Mat mat() const {
        return {q.data_ptr<uint8_t>(), scale.data_ptr<uint8_t>(), rows,
                block_rows};
    }
};

// checks what the kernels take for granted about a matrix given from outside
Blocks check_blocks(const Tensor& q, const Tensor& scale, int64_t cols,
                    int64_t block_rows, const char* name) {
    check_memory(q);
    check_memory(scale);
    TORCH_CHECK(!q.is_neg() && !scale.is_neg(), name,
                ": q and scale must be no negated views");
    TORCH_CHECK(q.is_cuda() && scale.device() == q.device(), name,
                ": q and scale must be on one GPU");
    TORCH_CHECK(q.scalar_type() == torch::kUInt8 &&
                    scale.scalar_type() == torch::kUInt8,
                name, ": q and scale must be uint8");
    TORCH_CHECK(block_rows == 1 || block_rows == 128, name,
                ": block_rows must be 1 or 128");
    TORCH_CHECK(cols >= 1 && cols <= (1 << 24), name,
                ": must have 1 to 2^24 columns");
    const int64_t nb = blocks_of(cols);
    TORCH_CHECK(q.dim() == 2 && q.size(1) == nb * 128 && q.is_contiguous(),
                name, ": q must be contiguous [rows, ", nb * 128, "]");
    TORCH_CHECK(q.size(0) <= (1 << 30), name, ": must have at most 2^30 rows");
    const int64_t sr =
        block_rows == 1 ? q.size(0) : (q.size(0) + 127) / 128;
    TORCH_CHECK(scale.dim() == 2 && scale.size(0) == sr &&
                    scale.size(1) == padded4(nb) && scale.is_contiguous(),
                name, ": scale must be contiguous [", sr, ", ", padded4(nb), "]");
    TORCH_CHECK(((uintptr_t)q.data_ptr() & 15) == 0 &&
                    ((uintptr_t)scale.data_ptr() & 3) == 0,
                name, ": q must be 16-byte and scale 4-byte aligned");
    return {q, scale, q.size(0), block_rows};
}

at::TensorOptions bytes_on(const Tensor& t) {
    return t.options().dtype(torch::kUInt8);
}
at::TensorOptions floats_on(const Tensor& t) {
    return t.options().dtype(torch::kFloat32);
}

// Workgroups that share out the rows: one for each pass of `rows_per_pass`
// rows, at most `most`.
int row_groups(int64_t rows, int64_t rows_per_pass, int64_t most) {
    return (int)std::min<int64_t>((rows + rows_per_pass - 1) / rows_per_pass,
                                  most);
}

Blocks new_blocks(const Tensor& like, int64_t R, int64_t C,
                  int64_t block_rows) {
    const int64_t nb = blocks_of(C);
    return {fresh({R, nb * 128}, bytes_on(like)),
            fresh({block_rows == 1 ? R : blocks_of(R), padded4(nb)},
                  bytes_on(like)),
            R, block_rows};
}

// workgroups of 4 waves that share out the rows of a strip of 4 blocks (or of
// 1, where there are fewer than 4)
int quant_groups(int64_t R, int64_t C, int64_t most) {
    return row_groups(R, blocks_of(C) >= 4 ? 4 : 16, most);
}

// Parts of one allocation: a training step of few rows is bound by the host,
// which each allocation costs 1.4 us and each tensor saved for the backward pass
// about as much.  [256, 1024, 3136]: 82 us a step, with 10 more of them 96.
struct Carve {
    int64_t size = 0;
    int64_t take(int64_t bytes) {
        const int64_t at = size;
        size += (bytes + 255) / 256 * 256;
        return at;
    }
    // a matrix [R, C]: where its bytes and its scales begin
    std::pair<int64_t, int64_t> matrix(int64_t R, int64_t C,
                                       int64_t block_rows) {
        const int64_t nb = blocks_of(C), q = take(R * nb * 128);
        return {q, take((block_rows == 1 ? R : blocks_of(R)) * padded4(nb))};
    }
};

Mat mat_at(uint8_t* base, std::pair<int64_t, int64_t> at, int64_t rows,
           int64_t block_rows) {
    return {base + at.first, base + at.second, rows, block_rows};
}

// Groups of rows for a quantisation that also sums up the columns: every group
// leaves a row of partial sums to be added up, and 1024 workgroups in all fill
// the card and keep those few.  More where a lane's register would add up over
// 256 rows, as far as a grid goes.
int sum_groups(int64_t R, int64_t C) {
    const int64_t nb = blocks_of(C), strips = nb >= 4 ? (nb + 3) / 4 : nb;
    const int64_t run = 256 * (nb >= 4 ? 4 : 16);  // a group's rows
    return quant_groups(
        R, C,
        std::min<int64_t>(65535, std::max<int64_t>({1, 1024 / strips,
                                                    (R + run - 1) / run})));
}

// scale per 1 x 128 block; with `mask` values whose bit is clear count as
// zero; `part` (may be null, [groups, C]) gets sums of the columns
void quant_rows(const Tensor& x, const uint8_t* mask, const Mat& o, float* part,
                int groups) {
    launched(riqn_fp8_quant_rows(x.data_ptr(),
                                 type_code(x.scalar_type(), "x"), x.stride(0),
                                 mask, o.q, o.scale, part, groups,
                                 (int)x.size(0), (int)x.size(1), stream_of(x)),
             "quantize_fp8_blocks");
}
Blocks quant_rows(const Tensor& x) {
    Blocks o = new_blocks(x, x.size(0), x.size(1), 1);
    quant_rows(x, nullptr, o.mat(), nullptr,
               quant_groups(x.size(0), x.size(1), 65535));
    return o;
}

void check_tiles(const Tensor& w) {
    TORCH_CHECK(blocks_of(w.size(0)) <= 65535 &&
                    blocks_of(w.size(0)) * blocks_of(w.size(1)) < (1 << 30),
                "a matrix with a scale per 128 x 128 block must have at most "
                "65535 blocks of rows and 2^30 blocks");
}

// scale per 128 x 128 block
Blocks quant_tiles(const Tensor& x) {
    check_tiles(x);
    Blocks o = new_blocks(x, x.size(0), x.size(1), 128);
    launched(riqn_fp8_quant_tiles(
                 x.data_ptr(), type_code(x.scalar_type(), "x"), x.stride(0),
                 o.q.data_ptr<uint8_t>(), o.scale.data_ptr<uint8_t>(), nullptr,
                 nullptr, (int)x.size(0), (int)x.size(1), stream_of(x)),
             "quantize_fp8_blocks");
    return o;
}

void gemm(const Mat& a, const Mat& b, int64_t K, const OptTensor& bias,
          bool relu, Tensor& c, uint8_t* mask, bool exact) {
    launched(riqn_fp8_gemm(
                 a.q, a.scale, (int)a.block_rows, b.q, b.scale,
                 (int)b.block_rows, bias ? bias->data_ptr() : nullptr,
                 bias ? type_code(bias->scalar_type(), "bias") : 0, relu,
                 c.data_ptr(), type_code(c.scalar_type(), "out"), mask, exact,
                 (int)a.rows, (int)b.rows, (int)K, stream_of(c)),
             "matmul_fp8_blocks");
}

std::tuple<Tensor, Tensor> fp8_blocks_quant(Tensor x, int64_t block_rows) {
    check_call();
    check_memory(x);
    x = x.resolve_neg();
    check_rows(x, "x");
    TORCH_CHECK(x.size(1) >= 1, "x must have at least one column");
    TORCH_CHECK(block_rows == 1 || block_rows == 128, "block_rows must be 1 or 128");
    type_code(x.scalar_type(), "x");
    c10::cuda::CUDAGuard guard(x.device());
    Blocks o = x.size(0) == 0    ? new_blocks(x, 0, x.size(1), block_rows)
               : block_rows == 1 ? quant_rows(x)
                                 : quant_tiles(x);
    return {o.q, o.scale};
}

Tensor fp8_blocks_dequant(Tensor q, Tensor scale, int64_t cols,
                          int64_t block_rows, at::ScalarType dtype) {
    check_call();
    Blocks b = check_blocks(q, scale, cols, block_rows, "blocks");
    const int type = type_code(dtype, "dtype");
    c10::cuda::CUDAGuard guard(q.device());
    Tensor out = fresh({b.rows, cols}, q.options().dtype(dtype));
    if (b.rows == 0) return out;
    launched(riqn_fp8_dequant(q.data_ptr<uint8_t>(), scale.data_ptr<uint8_t>(),
                              out.data_ptr(), type, (int)b.rows, (int)cols,
                              block_rows == 128 ? 7 : 0, stream_of(q)),
             "dequantize_fp8_blocks");
    return out;
}

Tensor fp8_blocks_matmul(Tensor aq, Tensor as, int64_t a_block_rows, Tensor bq,
                         Tensor bs, int64_t b_block_rows, int64_t cols,
                         OptTensor bias, bool relu, at::ScalarType dtype,
                         bool exact) {
    check_call();
    check_given(bias);
    Blocks a = check_blocks(aq, as, cols, a_block_rows, "a");
    Blocks b = check_blocks(bq, bs, cols, b_block_rows, "b");
    TORCH_CHECK(aq.device() == bq.device(), "a and b must be on one GPU");
    if (bias) {
        check_vector(*bias, b.rows, aq, "bias");
        type_code(bias->scalar_type(), "bias");
    }
    type_code(dtype, "out_dtype");
    c10::cuda::CUDAGuard guard(aq.device());
    Tensor c = fresh({a.rows, b.rows}, aq.options().dtype(dtype));
    if (c.numel() == 0) return c;
    gemm(a.mat(), b.mat(), cols, bias, relu, c, nullptr, exact);
    return c;
}

// x [..., C] as a matrix of contiguous rows, copied only where it must
Tensor as_rows(const Tensor& x) {
    Tensor r = x.resolve_neg();  // a view that negates is negated here
    if (x.dim() != 2) {
        TORCH_CHECK(x.dim() > 0, "a matrix or a vector is wanted, not a number");
        const int64_t c = x.size(-1);
        r = r.reshape({x.numel() / std::max<int64_t>(1, c), c});
    }
    return r.size(1) <= 1 || r.stride(1) == 1 ? r : r.contiguous();
}

std::vector<int64_t> with_last(const Tensor& x, int64_t n) {
    auto s = x.sizes().vec();
    s.back() = n;
    return s;
}

// y in another shape, but no view of y: a view that a custom function returns
// refuses to be changed in place
Tensor shaped(const Tensor& y, c10::IntArrayRef shape) {
    return y.sizes() == shape ? y : at::_unsafe_view(y, shape);
}

bool wants_grad(const Tensor& t) { return t.requires_grad(); }
bool wants_grad(const OptTensor& t) { return t && t->requires_grad(); }

// Gradients whose own gradients are not there: where a graph of the backward
// pass is being built, its use raises instead of counting as zero.
torch::autograd::variable_list once(torch::autograd::variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    torch::autograd::variable_list fake;
    for (auto& g : grads)
        fake.push_back(g.defined() ? g.detach().set_requires_grad(true) : g);
    auto err = std::make_shared<torch::autograd::DelayedError>(
        "this operator is differentiable once", (int)fake.size());
    return (*err)(std::move(fake));
}

// A gradient that goes on to a node of the default stream, such as a leaf's that
// a graph built outside the capture keeps alive, cannot be captured: the wait
// between the streams would break the capture and end the process.
void check_capture(const Tensor& t) {
    const auto stream = at::cuda::getCurrentCUDAStream(t.device().index());
    const c10::Stream other =
        at::cuda::getDefaultCUDAStream(t.device().index()).unwrap();
    if (stream.unwrap() == other) return;
    hipStreamCaptureStatus status;
    const hipError_t err = hipStreamIsCapturing(stream.stream(), &status);
    TORCH_CHECK(err == hipSuccess, hipGetErrorString(err));
    const auto node = torch::autograd::get_current_node();
    if (status == hipStreamCaptureStatusNone || !node) return;
    for (const auto& e : node->next_edges()) {
        if (!e.function) continue;
        const auto s = e.function->stream();
        TORCH_CHECK(!s || *s != other,
                    "a backward pass cannot be captured while a graph built on "
                    "the default stream is alive: drop its results first");
    }
}

// What waits for the backward pass, in one allocation: x in 8 bits; W
// transposed in 8 bits, for dx; the relu's bits.
struct Kept {
    std::pair<int64_t, int64_t> x, wt;
    int64_t bits, size;
    Kept(int64_t M, int64_t N, int64_t K, bool dx, bool relu) {
        Carve c;
        x = c.matrix(M, K, 1);
        if (dx) wt = c.matrix(K, N, 128);
        bits = c.take(relu ? M * blocks_of(N) * 16 : 0);
        size = c.size;
    }
};

// y = x W^T + bias, relu; `keep` gets what the backward pass reads (Kept)
Tensor linear_fwd(const Tensor& x, const Tensor& w, const OptTensor& bias,
                  bool relu, bool exact, bool need_dx, Tensor* keep) {
    check_rows(x, "x");
    check_rows(w, "weight");
    TORCH_CHECK(w.device() == x.device(), "weight must be on ", x.device());
    TORCH_CHECK(x.size(1) >= 1 && x.size(1) == w.size(1), "x has ", x.size(1),
                " columns and weight ", w.size(1));
    TORCH_CHECK(w.size(0) >= 1, "weight must have at least one row");
    if (bias) {
        check_vector(*bias, w.size(0), x, "bias");
        type_code(bias->scalar_type(), "bias");
    }
    const int type = type_code(x.scalar_type(), "x");
    const int w_type = type_code(w.scalar_type(), "weight");
    check_tiles(w);
    c10::cuda::CUDAGuard guard(x.device());
    const int64_t M = x.size(0), N = w.size(0), K = x.size(1);
    Tensor y = fresh({M, N}, x.options());
    if (M == 0 && !keep) return y;
    const Kept at(M, N, K, need_dx, relu && keep);
    Carve c;
    const auto w_at = c.matrix(N, K, 128);
    const int64_t x_at = c.take(keep ? 0 : at.size);
    Tensor work = fresh({c.size}, bytes_on(x));
    auto* const base = work.data_ptr<uint8_t>();
    if (keep) *keep = fresh({at.size}, bytes_on(x));
    auto* const kept = keep ? keep->data_ptr<uint8_t>() : base + x_at;
    const Mat xq = mat_at(kept, at.x, M, 1), wq = mat_at(base, w_at, N, 128);
    const Mat wt = need_dx ? mat_at(kept, at.wt, K, 128) : Mat{};
    const int groups = quant_groups(M, K, 65535);
    if (M > 0 && type == w_type) {
        launched(riqn_fp8_quant_both(x.data_ptr(), x.stride(0), xq.q, xq.scale,
                                     groups, (int)M, w.data_ptr(), w.stride(0),
                                     wq.q, wq.scale, wt.q, wt.scale, (int)N,
                                     (int)K, type, stream_of(x)),
                 "linear_fp8_blocks");
    } else {
        if (M > 0) quant_rows(x, nullptr, xq, nullptr, groups);
        launched(riqn_fp8_quant_tiles(w.data_ptr(), w_type, w.stride(0), wq.q,
                                      wq.scale, wt.q, wt.scale, (int)N, (int)K,
                                      stream_of(x)),
                 "linear_fp8_blocks");
    }
    if (M > 0)
        gemm(xq, wq, K, bias, relu, y, relu && keep ? kept + at.bits : nullptr,
             exact);
    return y;
}

struct LinearGrads {
    Tensor dx, dw, db;
};

// each gradient only where its dtype is given
LinearGrads linear_bwd(const Tensor& dy, const Tensor& keep, int64_t K, bool relu,
                       bool exact, c10::optional<at::ScalarType> dx_type,
                       c10::optional<at::ScalarType> dw_type,
                       c10::optional<at::ScalarType> db_type) {
    check_rows(dy, "dy");
    type_code(dy.scalar_type(), "dy");
    const int64_t M = dy.size(0), N = dy.size(1);
    const Kept at(M, N, K, dx_type.has_value(), relu);
    TORCH_CHECK(keep.device() == dy.device() && keep.size(0) == at.size,
                "dy does not have the result's rows or device");
    c10::cuda::CUDAGuard guard(dy.device());
    LinearGrads o;
    if (dx_type) o.dx = fresh({M, K}, dy.options().dtype(*dx_type));
    if (dw_type) o.dw = fresh({N, K}, dy.options().dtype(*dw_type));
    if (db_type) o.db = fresh({N}, dy.options().dtype(*db_type));
    if (M == 0) {
        if (dw_type) o.dw.zero_();
        if (db_type) o.db.zero_();
        return o;
    }
    // shares of the rows for each tile of 256 x 128 of dw: as many as two
    // workgroups a CU make one round of, with at least 256 rows each
    const int64_t tiles = (blocks_of(N) + 1) / 2 * blocks_of(K);
    const int shares = (int)std::max<int64_t>(
        1, std::min<int64_t>(std::min<int64_t>(512 / tiles, M / 256), 64));
    const int groups = db_type ? sum_groups(M, N) : quant_groups(M, N, 65535);
    Carve c;
    const auto g_at = c.matrix(M, N, 1);
    const int64_t sum_at = c.take(db_type ? groups * N * 4 : 0);
    const int64_t part_at = c.take(dw_type && shares > 1 ? shares * N * K * 4 : 0);
    Tensor work = fresh({c.size}, bytes_on(dy));
    auto* const base = work.data_ptr<uint8_t>();
    auto* const kept = keep.data_ptr<uint8_t>();
    const Mat g = mat_at(base, g_at, M, 1), x = mat_at(kept, at.x, M, 1);
    float* const sums = db_type ? (float*)(base + sum_at) : nullptr;
    quant_rows(dy, relu ? kept + at.bits : nullptr, g, sums, groups);
    if (db_type)
        launched(riqn_column_sum(sums, o.db.data_ptr(),
                                 type_code(*db_type, "bias"), groups, (int)N,
                                 stream_of(dy)),
                 "column sum");
    if (dx_type)
        gemm(g, mat_at(kept, at.wt, K, 128), N, c10::nullopt, false, o.dx,
             nullptr, exact);
    if (dw_type)
        launched(riqn_fp8_wgrad(
                     g.q, g.scale, x.q, x.scale, o.dw.data_ptr(),
                     type_code(*dw_type, "weight"),
                     shares > 1 ? (float*)(base + part_at) : nullptr, shares,
                     (int)M, (int)N, (int)K, stream_of(dy)),
                 "linear_fp8_blocks backward");
    return o;
}

// Autograd in C++: a training step of a small batch is bound by the host, and
// a Python autograd function costs more than its kernels.
class LinearFn : public torch::autograd::Function<LinearFn> {
  public:
    static Tensor forward(torch::autograd::AutogradContext* ctx, Tensor x,
                          Tensor w, OptTensor bias, bool relu, bool exact,
                          bool ndx, bool ndw, bool ndb) {
        Tensor keep;
        Tensor y =
            linear_fwd(as_rows(x), as_rows(w), bias, relu, exact, ndx, &keep);
        ctx->save_for_backward({keep});
        // the relu, exactness, the types of the gradients, then x's shape
        std::vector<int64_t> d = {
            relu, exact, ndx ? (int64_t)x.scalar_type() : -1,
            ndw ? (int64_t)w.scalar_type() : -1,
            ndb ? (int64_t)bias->scalar_type() : -1};
        d.insert(d.end(), x.sizes().begin(), x.sizes().end());
        ctx->saved_data["all"] = std::move(d);
        return shaped(y, with_last(x, w.size(0)));
    }
    static torch::autograd::variable_list backward(
        torch::autograd::AutogradContext* ctx,
        torch::autograd::variable_list dy) {
        check_given(dy[0]);
        check_capture(dy[0]);
        const auto v = ctx->get_saved_variables();
        const auto d = ctx->saved_data["all"].toIntVector();
        auto type = [&](int i) -> c10::optional<at::ScalarType> {
            if (d[i] < 0) return c10::nullopt;
            return (at::ScalarType)d[i];
        };
        LinearGrads g = linear_bwd(as_rows(dy[0]), v[0], d.back(), d[0], d[1],
                                   type(2), type(3), type(4));
        if (g.dx.defined())
            g.dx = shaped(g.dx, c10::IntArrayRef(d).slice(5));
        return once({g.dx, g.dw, g.db, Tensor(), Tensor(), Tensor(), Tensor(),
                     Tensor()});
    }
};

Tensor linear_fp8(Tensor x, Tensor w, OptTensor bias, bool relu, bool exact) {
    check_call();
    check_given(x);
    check_given(w);
    check_given(bias);
    TORCH_CHECK(w.dim() == 2, "weight must have 2 dimensions");
    if (!at::GradMode::is_enabled() ||
        !(wants_grad(x) || wants_grad(w) || wants_grad(bias)))
        return shaped(linear_fwd(as_rows(x), as_rows(w), bias, relu, exact,
                                 false, nullptr),
                      with_last(x, w.size(0)));
    return LinearFn::apply(x, w, bias, relu, exact, wants_grad(x), wants_grad(w),
                           wants_grad(bias));
}

// the same against a weight that is in 8 bits already; no gradients
Tensor linear_fp8_serve(Tensor x0, Tensor wq, Tensor ws, int64_t block_rows,
                        OptTensor bias, bool relu, bool exact) {
    TORCH_CHECK(!at::GradMode::is_enabled() ||
                    !(wants_grad(x0) || wants_grad(bias)),
                "a weight in 8-bit blocks is for serving: pass the float "
                "weight where gradients are wanted");
    check_call();
    check_given(x0);
    check_given(bias);
    const Tensor x = as_rows(x0);
    check_rows(x, "x");
    Blocks w = check_blocks(wq, ws, x.size(1), block_rows, "weight");
    TORCH_CHECK(wq.device() == x.device(), "weight must be on ", x.device());
    if (bias) {
        check_vector(*bias, w.rows, x, "bias");
        type_code(bias->scalar_type(), "bias");
    }
    type_code(x.scalar_type(), "x");
    c10::cuda::CUDAGuard guard(x.device());
    Tensor y = fresh({x.size(0), w.rows}, x.options());
    if (y.numel() > 0 && riqn_fp8_few(x.size(0), w.rows, (int)x.size(1)))
        launched(riqn_fp8_gemm_from(
                     x.data_ptr(), type_code(x.scalar_type(), "x"), x.stride(0),
                     w.q.data_ptr<uint8_t>(), w.scale.data_ptr<uint8_t>(),
                     (int)block_rows, bias ? bias->data_ptr() : nullptr,
                     bias ? type_code(bias->scalar_type(), "bias") : 0, relu,
                     y.data_ptr(), (int)x.size(0), (int)w.rows, (int)x.size(1),
                     stream_of(x)),
                 "linear_fp8_blocks");
    else if (y.numel() > 0)
        gemm(quant_rows(x).mat(), w.mat(), x.size(1), bias, relu, y, nullptr,
             exact);
    return shaped(y, with_last(x0, w.rows));
}

int norm_weights(const Tensor& x, const OptTensor& w, const OptTensor& b) {
    const int xt = type_code(x.scalar_type(), "x");
    int wt = -1;
    for (const auto* t : {&w, &b}) {
        if (!*t) continue;
        check_vector(**t, x.size(1), x, "weight and bias");
        const int code = type_code((*t)->scalar_type(), "weight and bias");
        TORCH_CHECK(code == xt || code == 0,
                    "weight and bias must have x's dtype or float32");
        TORCH_CHECK(wt < 0 || wt == code, "weight and bias must have one dtype");
        wt = code;
    }
    return wt < 0 ? xt : wt;
}

// stats gets each row's mean, then each row's rstd; null where no backward pass
// will ask for them
Tensor norm_fwd(const Tensor& x, const OptTensor& w, const OptTensor& b,
                double eps, Tensor* stats) {
    check_rows(x, "x");
    TORCH_CHECK(x.size(1) >= 1, "x must have at least one column");
    TORCH_CHECK(eps >= 0.0, "eps must not be negative");
    const int wt = norm_weights(x, w, b);
    c10::cuda::CUDAGuard guard(x.device());
    Tensor y = fresh({x.size(0), x.size(1)}, x.options());
    float* mean = nullptr;
    if (stats) {
        *stats = fresh({2 * x.size(0)}, floats_on(x));
        mean = stats->data_ptr<float>();
    }
    if (x.size(0) > 0)
        launched(riqn_norm_fwd(
                     x.data_ptr(), type_code(x.scalar_type(), "x"), x.stride(0),
                     w ? w->data_ptr() : nullptr, b ? b->data_ptr() : nullptr,
                     wt, y.data_ptr(), mean, mean ? mean + x.size(0) : nullptr,
                     (int)x.size(0), (int)x.size(1), (float)eps, stream_of(x)),
                 "layer_norm");
    return y;
}

class NormFn : public torch::autograd::Function<NormFn> {
  public:
    static Tensor forward(torch::autograd::AutogradContext* ctx, Tensor x,
                          OptTensor w, OptTensor b, double eps, bool ndx,
                          bool ndw, bool ndb) {
        const Tensor x2 = as_rows(x);
        Tensor stats;
        Tensor y = norm_fwd(x2, w, b, eps, &stats);
        ctx->save_for_backward({x2, w ? *w : Tensor(), stats});
        // which gradients, their type, then x's shape
        std::vector<int64_t> d = {ndx | ndw << 1 | ndb << 2,
                                  (int64_t)(w ? *w : b ? *b : x).scalar_type()};
        d.insert(d.end(), x.sizes().begin(), x.sizes().end());
        ctx->saved_data["all"] = std::move(d);
        return shaped(y, x.sizes());
    }
    static torch::autograd::variable_list backward(
        torch::autograd::AutogradContext* ctx,
        torch::autograd::variable_list grad) {
        check_given(grad[0]);
        check_capture(grad[0]);
        const auto v = ctx->get_saved_variables();
        const Tensor &x = v[0], &w = v[1];
        check_rows(x, "x");
        TORCH_CHECK(v[2].device() == x.device() &&
                        (!w.defined() || w.device() == x.device()),
                    "what was kept must be on one GPU");
        const float* const mean = v[2].data_ptr<float>();
        const auto d = ctx->saved_data["all"].toIntVector();
        const int64_t need = d[0];
        const auto w_type = (at::ScalarType)d[1];
        const Tensor dy = as_rows(grad[0]);
        TORCH_CHECK(dy.sizes() == x.sizes() && dy.device() == x.device() &&
                        dy.scalar_type() == x.scalar_type(),
                    "dy must have x's shape, device and dtype");
        const int64_t R = x.size(0), C = x.size(1);
        c10::cuda::CUDAGuard guard(x.device());
        Tensor dx, dw, db;
        if (need & 1) dx = fresh({R, C}, x.options());
        if (need & 2) dw = fresh({C}, x.options().dtype(w_type));
        if (need & 4) db = fresh({C}, x.options().dtype(w_type));
        if (R == 0) {
            if (dw.defined()) dw.zero_();
            if (db.defined()) db.zero_();
        } else {
            const int groups = riqn_norm_groups((int)R, (int)C);
            Tensor part;
            if (need & 6) part = fresh({groups, 2, C}, floats_on(x));
            launched(riqn_norm_bwd(
                         dy.data_ptr(), x.data_ptr(),
                         type_code(x.scalar_type(), "x"), dy.stride(0),
                         x.stride(0), w.defined() ? w.data_ptr() : nullptr,
                         type_code(w_type, "weight"), mean, mean + R,
                         need & 1 ? dx.data_ptr() : nullptr,
                         need & 2 ? dw.data_ptr() : nullptr,
                         need & 4 ? db.data_ptr() : nullptr,
                         need & 6 ? part.data_ptr<float>() : nullptr, groups,
                         (int)R, (int)C, stream_of(x)),
                     "layer_norm backward");
        }
        if (need & 1) dx = shaped(dx, c10::IntArrayRef(d).slice(2));
        return once({dx, dw, db, Tensor(), Tensor(), Tensor(), Tensor()});
    }
};

Tensor layer_norm(Tensor x, OptTensor w, OptTensor b, double eps) {
    check_call();
    check_given(x);
    check_given(w);
    check_given(b);
    if (!at::GradMode::is_enabled() ||
        !(wants_grad(x) || wants_grad(w) || wants_grad(b)))
        return shaped(norm_fwd(as_rows(x), w, b, eps, nullptr), x.sizes());
    return NormFn::apply(x, w, b, eps, wants_grad(x), wants_grad(w),
                         wants_grad(b));
}

}  // namespace

void bind_blocks(py::module& m) {
    m.def("fp8_blocks_quant", &fp8_blocks_quant);
    m.def("fp8_blocks_dequant", &fp8_blocks_dequant);
    m.def("fp8_blocks_matmul", &fp8_blocks_matmul);
    m.def("linear_fp8", &linear_fp8);
    m.def("linear_fp8_serve", &linear_fp8_serve);
    m.def("layer_norm", &layer_norm);
}
