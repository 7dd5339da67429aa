// The hot torch.ops.npu.* kernels in C++: argument checks, output allocation and
// the C ABI call, without Python between the dispatcher and the launch.
//
// An op called from Python used to spend 15-25 us in its Python kernel (checks,
// three tensor allocations, ctypes), more than the launches of a decode-sized
// linear take on the GPU; here the same steps take 3-5 us (one row of a 5120 x 5120
// linear module 22 -> 7.7 us per call, the GPU's share 7.4).
//
// Schemas, fake kernels and the remaining ops stay in ops.py, the checks and their
// messages are those of the Python kernels these replace (TORCH_CHECK raises
// RuntimeError).  The C ABI library is not linked: its entry points are asked for
// once, at the first call, through the Python loader (_abi.lib(), which honours
// W4A8_AMD_LIB and raises FileNotFoundError where the library is missing), and
// workspaces come from ops._workspace, which keeps one per device and stream and
// per graph capture.
#define __HIP_PLATFORM_AMD__ 1
#include <torch/extension.h>

#include <c10/hip/HIPStream.h>

#include <array>
#include <atomic>
#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "../../include/w4a8_amd.h"
#include "kgeom.h"

namespace {

namespace geom = w4a8::geom;
using at::Tensor;

// The C ABI entry points used here, in the order bind() receives their addresses.
#define W4A8_TORCH_FNS(F)                                                                                     \
    F(w4a8_last_error) F(w4a8_quant_act) F(w4a8_gemm_workspace_bytes) F(w4a8_gemm) F(w4a8_gemm_swiglu)        \
    F(w4a8_linear_bias) F(w4a8_rmsnorm_quant) F(w4a8_rope_kv) F(w4a8_attention) F(w4a8_attention_rope)        \
    F(w4a8_attention_workspace_bytes) F(w4a8_rope_kv8) F(w4a8_kv8_read) F(w4a8_attention_kv8)                 \
    F(w4a8_attention_kv8_rope) F(w4a8_attention_kv8_workspace_bytes) F(w4a8_midgroup_quant_a)                 \
    F(w4a8_midgroup_gemm_workspace_bytes)                                                                     \
    F(w4a8_midgroup_split_workspace_bytes) F(w4a8_midgroup_gemm_split) F(w4a8_midgroup_tiles_bytes)           \
    F(w4a8_midgroup_gemm_ws) F(w4a8_midgroup_gemm_tiled)

struct Abi {
#define W4A8_DECL(n) decltype(&::n) n;
    W4A8_TORCH_FNS(W4A8_DECL)
#undef W4A8_DECL
};

std::vector<std::string> abi_names() {
    return {
#define W4A8_NAME(n) #n,
        W4A8_TORCH_FNS(W4A8_NAME)
#undef W4A8_NAME
    };
}

// Set once from Python at import; never destroyed (the interpreter may be gone first).
PyObject* g_loader = nullptr;      // () -> addresses of abi_names()
PyObject* g_workspace = nullptr;   // (device index, bytes) -> (address, bytes)
Abi g_abi;
std::atomic<bool> g_bound{false};

const Abi& abi() {
    if (!g_bound.load(std::memory_order_acquire)) {
        py::gil_scoped_acquire gil;   // also serialises the first calls of several threads
        if (!g_bound.load(std::memory_order_relaxed)) {
            TORCH_CHECK(g_loader != nullptr, "w4a8: the torch layer is not initialised");
            const auto a = py::reinterpret_borrow<py::object>(g_loader)().cast<std::vector<uintptr_t>>();
            size_t i = 0;
#define W4A8_SET(n) g_abi.n = reinterpret_cast<decltype(&::n)>(a.at(i++));
            W4A8_TORCH_FNS(W4A8_SET)
#undef W4A8_SET
            g_bound.store(true, std::memory_order_release);
        }
    }
    return g_abi;
}

void check(int status, const char* what) {
    if (status == 0) return;
    static const char* const names[] = {"OK", "NULL", "SHAPE", "DTYPE", "ALIGN", "UNSUPPORTED", "WORKSPACE", "HIP"};
    const std::string name = status > 0 && status < 8 ? names[status] : std::to_string(status);
    TORCH_CHECK(false, what, " failed (", name, "): ", abi().w4a8_last_error());
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

struct Workspace {
    void* ptr = nullptr;
    int64_t bytes = 0;
};

Workspace workspace(const Tensor& t, int64_t need) {
    py::gil_scoped_acquire gil;
    const auto r = py::reinterpret_borrow<py::object>(g_workspace)(static_cast<int>(t.device().index()), need)
                       .cast<std::pair<uintptr_t, int64_t>>();
    return {reinterpret_cast<void*>(r.first), r.second};
}

Tensor empty(at::IntArrayRef sizes, at::ScalarType dt, const Tensor& like) {
    return at::empty(sizes, at::TensorOptions().dtype(dt).device(like.device()));
}

// A tensor whose rows are contiguous (and row starts a multiple of `align` elements apart).
Tensor rows(const Tensor& t, int64_t align = 1) {
    return t.stride(1) != 1 || t.stride(0) % align ? t.contiguous() : t;
}

const void* opt_ptr(const std::optional<Tensor>& t) { return t.has_value() ? t->data_ptr() : nullptr; }

bool is_scale(at::ScalarType t) { return t == at::kHalf || t == at::kBFloat16; }
int scale_code(const Tensor& t) { return t.scalar_type() == at::kBFloat16 ? W4A8_DT_BF16 : W4A8_DT_F16; }

// Python's floor-based integer arithmetic is not needed: K and group are checked positive
// where the geometry divides by them.
void check_geometry(const char* op, int64_t K, int64_t group) {
    TORCH_CHECK(K > 0 && group > 0, op, ": K=", K, " and group=", group, " must be > 0");
}

int64_t quant_width(int64_t K, int64_t group) { return group > 0 && K > 0 ? geom::kpad(K, group) : K; }

// ------------------------------------------------------------------ quant
std::tuple<Tensor, Tensor> quant_pertoken(const Tensor& x0, int64_t group) {
    TORCH_CHECK(x0.dim() == 2, "w4a8_quant_pertoken: x must be [M, K]");
    TORCH_CHECK(x0.scalar_type() == at::kBFloat16, "w4a8_quant_pertoken: x must be bfloat16");
    TORCH_CHECK(group >= 0, "w4a8_quant_pertoken: group must be >= 0");
    const Tensor x = rows(x0);
    const int64_t M = x.size(0), K = x.size(1), width = quant_width(K, group);
    Tensor a_q = empty({M, width}, at::kChar, x), a_scale = empty({M}, at::kBFloat16, x);
    if (M)
        check(abi().w4a8_quant_act(x.data_ptr(), x.stride(0), a_q.data_ptr(), width, a_scale.data_ptr(), M, K, group,
                                   stream_of(x)),
              "w4a8_quant_pertoken");
    return {a_q, a_scale};
}

// ------------------------------------------------------------------ gemm
void check_weights(const Tensor& w_tiles, const Tensor& s_tiles, int64_t N, int64_t K, int64_t group) {
    TORCH_CHECK(w_tiles.scalar_type() == at::kByte &&
                    w_tiles.numel() == geom::col_blocks(N) * geom::k_tiles(K, group) * geom::kTileBytes,
                "w4a8_gemm: w_tiles must be the uint8 output of w4a8_repack for (N, K, group)");
    TORCH_CHECK(is_scale(s_tiles.scalar_type()) && s_tiles.dim() == 3 && s_tiles.size(0) == geom::col_blocks(N) &&
                    s_tiles.size(1) == geom::num_groups(K, group) && s_tiles.size(2) == geom::kTileN,
                "w4a8_gemm: s_tiles must be the scale output of w4a8_repack for (N, K, group)");
}

Tensor run_gemm(const Tensor& a_q0, const Tensor& a_scale0, const Tensor& w_tiles, const Tensor& s_tiles, int64_t N,
                int64_t K, int64_t group, bool swiglu) {
    check_geometry("w4a8_gemm", K, group);
    const int64_t kpad = geom::kpad(K, group);
    TORCH_CHECK(a_q0.dim() == 2 && a_q0.scalar_type() == at::kChar, "w4a8_gemm: a_q must be int8 [M, kpad]");
    TORCH_CHECK(a_q0.size(1) == kpad, "w4a8_gemm: a_q has ", a_q0.size(1),
                " columns; the padded group layout of K=", K, ", group=", group, " has ", kpad,
                " (w4a8_quant_pertoken(x, group))");
    TORCH_CHECK(a_scale0.scalar_type() == at::kBFloat16 && a_scale0.dim() == 1 && a_scale0.size(0) == a_q0.size(0),
                "w4a8_gemm: a_scale must be bfloat16 [M]");
    check_weights(w_tiles, s_tiles, N, K, group);
    TORCH_CHECK(!swiglu || N % 32 == 0, "w4a8_gemm_swiglu: N=", N, " must be 2*I with I a multiple of 16");
    const Tensor a_q = rows(a_q0, 16), a_scale = a_scale0.contiguous();
    const int64_t M = a_q.size(0), ncols = swiglu ? N / 2 : N;
    Tensor y = empty({M, ncols}, at::kBFloat16, a_q);
    if (M == 0) return y;
    const Abi& f = abi();
    const int64_t need = f.w4a8_gemm_workspace_bytes(M, N, K, group);
    const Workspace ws = need > 0 ? workspace(a_q, need) : Workspace{};
    check((swiglu ? f.w4a8_gemm_swiglu : f.w4a8_gemm)(a_q.data_ptr(), a_q.stride(0), a_scale.data_ptr(),
                                                      w_tiles.data_ptr(), s_tiles.data_ptr(), scale_code(s_tiles),
                                                      y.data_ptr(), ncols, M, N, K, group, ws.ptr, ws.bytes,
                                                      stream_of(a_q)),
          "w4a8_gemm");
    return y;
}

Tensor gemm(const Tensor& a_q, const Tensor& a_scale, const Tensor& w_tiles, const Tensor& s_tiles, int64_t N,
            int64_t K, int64_t group) {
    return run_gemm(a_q, a_scale, w_tiles, s_tiles, N, K, group, false);
}

Tensor gemm_swiglu(const Tensor& a_q, const Tensor& a_scale, const Tensor& w_tiles, const Tensor& s_tiles, int64_t N,
                   int64_t K, int64_t group) {
    return run_gemm(a_q, a_scale, w_tiles, s_tiles, N, K, group, true);
}

// ------------------------------------------------------------------ quant + GEMM
Tensor linear(const Tensor& x0, const Tensor& w_tiles, const Tensor& s_tiles, int64_t N, int64_t K, int64_t group,
              const std::optional<Tensor>& bias0) {
    TORCH_CHECK(x0.dim() == 2 && x0.scalar_type() == at::kBFloat16, "w4a8_linear: x must be bfloat16 [M, K]");
    TORCH_CHECK(x0.size(1) == K, "w4a8_linear: x has ", x0.size(1), " columns, K=", K);
    check_geometry("w4a8_linear", K, group);
    check_weights(w_tiles, s_tiles, N, K, group);
    std::optional<Tensor> bias;
    if (bias0.has_value()) {
        TORCH_CHECK(bias0->scalar_type() == at::kBFloat16 && bias0->dim() == 1 && bias0->size(0) == N &&
                        bias0->device() == x0.device(),
                    "w4a8_linear: bias must be bfloat16 [N] on the device of x");
        bias = bias0->contiguous();
    }
    const Tensor x = rows(x0);
    const int64_t M = x.size(0), width = geom::kpad(K, group);
    Tensor y = empty({M, N}, at::kBFloat16, x);
    if (M == 0) return y;
    // one scratch tensor: the int8 rows, then the bf16 scales
    const int64_t as_off = (M * width + 255) / 256 * 256;
    const Tensor aq = empty({as_off + 2 * M}, at::kChar, x);
    char* const p = static_cast<char*>(aq.data_ptr());
    const Abi& f = abi();
    // the prefill kernels' epilogue adds the bias; up to kDecodeMaxM rows torch does
    const bool epilogue = bias.has_value() && M > w4a8::kDecodeMaxM;
    const int64_t need = f.w4a8_gemm_workspace_bytes(M, N, K, group);
    const Workspace ws = need > 0 ? workspace(x, need) : Workspace{};
    check(f.w4a8_linear_bias(x.data_ptr(), x.stride(0), w_tiles.data_ptr(), s_tiles.data_ptr(), scale_code(s_tiles),
                             epilogue ? bias->data_ptr() : nullptr, y.data_ptr(), N, p, width, p + as_off, M, N, K,
                             group, ws.ptr, ws.bytes, stream_of(x)),
          "w4a8_linear");
    if (bias.has_value() && !epilogue) {
        at::AutoDispatchBelowADInplaceOrView guard;   // the op has no derivative, with any row count
        y.add_(*bias);
    }
    return y;
}

// ------------------------------------------------------------------ RMSNorm + quant
std::tuple<Tensor, Tensor, Tensor, Tensor> rmsnorm_quant(const Tensor& x0, const Tensor& weight0, double eps,
                                                         const std::optional<Tensor>& residual0, int64_t group,
                                                         bool want_normed) {
    TORCH_CHECK(x0.dim() == 2 && x0.scalar_type() == at::kBFloat16, "w4a8_rmsnorm_quant: x must be bfloat16 [M, K]");
    const int64_t M = x0.size(0), K = x0.size(1);
    TORCH_CHECK(weight0.scalar_type() == at::kBFloat16 && weight0.dim() == 1 && weight0.size(0) == K,
                "w4a8_rmsnorm_quant: weight must be bfloat16 [K]");
    const Tensor x = rows(x0, 8), weight = weight0.contiguous();
    Tensor residual, s;
    if (residual0.has_value()) {
        TORCH_CHECK(residual0->scalar_type() == at::kBFloat16 && residual0->sizes() == x.sizes(),
                    "w4a8_rmsnorm_quant: residual must match x");
        residual = rows(*residual0, 8);
        s = at::empty_like(x);
    } else {
        s = empty({0, K}, at::kBFloat16, x);
    }
    const int64_t width = quant_width(K, group);
    Tensor a_q = empty({M, width}, at::kChar, x), a_scale = empty({M}, at::kBFloat16, x);
    Tensor h = empty({want_normed ? M : 0, K}, at::kBFloat16, x);
    if (M)
        check(abi().w4a8_rmsnorm_quant(x.data_ptr(), x.stride(0), residual.defined() ? residual.data_ptr() : nullptr,
                                       residual.defined() ? residual.stride(0) : 0, weight.data_ptr(),
                                       static_cast<float>(eps), residual.defined() ? s.data_ptr() : nullptr, K,
                                       want_normed ? h.data_ptr() : nullptr, K, a_q.data_ptr(), width,
                                       a_scale.data_ptr(), M, K, group, stream_of(x)),
              "w4a8_rmsnorm_quant");
    return {a_q, a_scale, s, h};
}

// ------------------------------------------------------------------ RoPE + KV-cache append
void check_tables(const char* op, const Tensor& cos, const Tensor& sin, int64_t L, int64_t D) {
    for (const auto& [t, name] : {std::pair<const Tensor&, const char*>{cos, "cos"}, {sin, "sin"}})
        TORCH_CHECK(t.dim() == 2 && t.scalar_type() == at::kFloat && t.size(0) >= L && t.size(1) >= D / 2 &&
                        t.stride(1) == 1,
                    op, ": ", name, " must be float32 [>= L, >= head_dim / 2]");
    TORCH_CHECK(cos.stride(0) == sin.stride(0), op, ": cos and sin must share a row stride");
}

std::optional<Tensor> check_bias(const char* op, const std::optional<Tensor>& bias, int64_t W, const Tensor& qkv) {
    if (!bias.has_value()) return std::nullopt;
    TORCH_CHECK(bias->scalar_type() == at::kBFloat16 && bias->numel() == W && bias->device() == qkv.device(), op,
                ": bias must be bfloat16 [(heads + 2 kv_heads) * head_dim] on the device");
    return bias->contiguous();
}

Tensor rope_kv(const Tensor& qkv0, const Tensor& cos, const Tensor& sin, const Tensor& pos, const Tensor& k_cache,
               const Tensor& v_cache, int64_t heads, int64_t kv_heads, const std::optional<Tensor>& bias0) {
    TORCH_CHECK(qkv0.dim() == 3 && qkv0.scalar_type() == at::kBFloat16, "w4a8_rope_kv: qkv must be bfloat16 [B, T, W]");
    const int64_t B = qkv0.size(0), T = qkv0.size(1), W = qkv0.size(2);
    TORCH_CHECK(heads > 0 && kv_heads > 0 && W % (heads + 2 * kv_heads) == 0,
                "w4a8_rope_kv: qkv width must be (heads + 2 kv_heads) * head_dim");
    const int64_t D = W / (heads + 2 * kv_heads);
    TORCH_CHECK(D % 2 == 0, "w4a8_rope_kv: head_dim must be even");
    TORCH_CHECK(k_cache.dim() == 4 && v_cache.dim() == 4 && k_cache.scalar_type() == at::kBFloat16 &&
                    v_cache.scalar_type() == at::kBFloat16,
                "w4a8_rope_kv: caches must be 4-D bfloat16");
    const int64_t L = k_cache.size(3);
    TORCH_CHECK(k_cache.sizes() == at::IntArrayRef({B, kv_heads, D, L}) &&
                    v_cache.sizes() == at::IntArrayRef({B, kv_heads, L, D}),
                "w4a8_rope_kv: caches must be k [B, kv_heads, D, L] and v [B, kv_heads, L, D]");
    check_tables("w4a8_rope_kv", cos, sin, L, D);
    TORCH_CHECK(pos.scalar_type() == at::kLong && pos.numel() == 1 && pos.device() == qkv0.device(),
                "w4a8_rope_kv: pos must be one int64 on the device (the position of token 0, shared by every "
                "sequence; per-sequence positions are not supported)");
    const Tensor qkv = qkv0.stride(2) != 1 || qkv0.stride(0) != T * qkv0.stride(1) ? qkv0.contiguous() : qkv0;
    const auto bias = check_bias("w4a8_rope_kv", bias0, W, qkv);
    Tensor q = empty({B, T, heads, D}, at::kBFloat16, qkv);
    if (B * T)
        check(abi().w4a8_rope_kv(qkv.data_ptr(), qkv.stride(1), opt_ptr(bias), cos.data_ptr(), sin.data_ptr(),
                                 cos.stride(0), L, pos.data_ptr(), q.data_ptr(), k_cache.data_ptr(),
                                 k_cache.strides().data(), v_cache.data_ptr(), v_cache.strides().data(), B, T, heads,
                                 kv_heads, D, stream_of(qkv)),
              "w4a8_rope_kv");
    return q;
}

// ------------------------------------------------------------------ attention
float softmax_scale(const std::optional<double>& scale, int64_t D) {
    return static_cast<float>(scale.has_value() ? *scale : 1.0 / std::sqrt(static_cast<double>(D)));
}

Tensor attention(const Tensor& q0, const Tensor& k_cache, const Tensor& vt_cache, const Tensor& pos, int64_t L,
                 int64_t cps, bool split, const std::optional<double>& scale) {
    TORCH_CHECK(q0.dim() == 4 && q0.scalar_type() == at::kBFloat16, "w4a8_attention: q must be bfloat16 [B, T, H, D]");
    const int64_t B = q0.size(0), T = q0.size(1), H = q0.size(2), D = q0.size(3);
    TORCH_CHECK(k_cache.dim() == 4 && vt_cache.dim() == 4 && k_cache.scalar_type() == at::kBFloat16 &&
                    vt_cache.scalar_type() == at::kBFloat16,
                "w4a8_attention: caches must be 4-D bfloat16");
    const int64_t KVH = k_cache.size(1), Lc = k_cache.size(2);
    TORCH_CHECK(k_cache.sizes() == at::IntArrayRef({B, KVH, Lc, D}) &&
                    vt_cache.sizes() == at::IntArrayRef({B, KVH, D, Lc}),
                "w4a8_attention: caches must be k [B, kv_heads, Lc, D] and vt [B, kv_heads, D, Lc]");
    TORCH_CHECK(k_cache.is_contiguous() && vt_cache.is_contiguous(), "w4a8_attention: caches must be contiguous");
    TORCH_CHECK(pos.scalar_type() == at::kLong && pos.numel() == 1 && pos.device() == q0.device(),
                "w4a8_attention: pos must be one int64 on the device");
    const Tensor q = q0.contiguous();
    Tensor out = at::empty_like(q);
    if (B * T == 0) return out;
    const Abi& f = abi();
    Workspace ws;
    if (split) {
        const int64_t need = f.w4a8_attention_workspace_bytes(B, T, H, D, Lc, cps);
        TORCH_CHECK(need >= 0, "w4a8_attention: bad shape for the workspace size");
        ws = workspace(q, std::max<int64_t>(need, 16));
    }
    check(f.w4a8_attention(q.data_ptr(), k_cache.data_ptr(), vt_cache.data_ptr(), out.data_ptr(), pos.data_ptr(), B, T,
                           H, KVH, D, L, Lc, cps, softmax_scale(scale, D), ws.ptr, ws.bytes, stream_of(q)),
          "w4a8_attention");
    return out;
}

Tensor attention_rope(const Tensor& qkv0, const Tensor& cos, const Tensor& sin, const Tensor& pos,
                      const Tensor& k_cache, const Tensor& vt_cache, int64_t heads, int64_t kv_heads, int64_t L,
                      int64_t cps, const std::optional<Tensor>& bias0, const std::optional<double>& scale) {
    TORCH_CHECK(qkv0.dim() == 2 && qkv0.scalar_type() == at::kBFloat16,
                "w4a8_attention_rope: qkv must be bfloat16 [B, W]");
    const int64_t B = qkv0.size(0), W = qkv0.size(1);
    TORCH_CHECK(heads > 0 && kv_heads > 0 && W % (heads + 2 * kv_heads) == 0,
                "w4a8_attention_rope: qkv width must be (heads + 2 kv_heads) * head_dim");
    const int64_t D = W / (heads + 2 * kv_heads);
    TORCH_CHECK(k_cache.dim() == 4 && vt_cache.dim() == 4 && k_cache.scalar_type() == at::kBFloat16 &&
                    vt_cache.scalar_type() == at::kBFloat16,
                "w4a8_attention_rope: caches must be 4-D bfloat16");
    const int64_t Lc = k_cache.size(2);
    TORCH_CHECK(k_cache.sizes() == at::IntArrayRef({B, kv_heads, Lc, D}) &&
                    vt_cache.sizes() == at::IntArrayRef({B, kv_heads, D, Lc}) && k_cache.is_contiguous() &&
                    vt_cache.is_contiguous(),
                "w4a8_attention_rope: caches must be contiguous k [B, kv_heads, Lc, D] and vt [B, kv_heads, D, Lc]");
    check_tables("w4a8_attention_rope", cos, sin, L, D);
    TORCH_CHECK(pos.scalar_type() == at::kLong && pos.numel() == 1 && pos.device() == qkv0.device(),
                "w4a8_attention_rope: pos must be one int64 on the device");
    const Tensor qkv = rows(qkv0, 8);
    const auto bias = check_bias("w4a8_attention_rope", bias0, W, qkv);
    Tensor out = empty({B, 1, heads, D}, at::kBFloat16, qkv);
    if (B == 0) return out;
    const Abi& f = abi();
    const int64_t need = f.w4a8_attention_workspace_bytes(B, 1, heads, D, Lc, cps);
    TORCH_CHECK(need >= 0, "w4a8_attention_rope: bad shape for the workspace size");
    const Workspace ws = need > 0 ? workspace(qkv, need) : Workspace{};
    check(f.w4a8_attention_rope(qkv.data_ptr(), qkv.stride(0), opt_ptr(bias), cos.data_ptr(), sin.data_ptr(),
                                cos.stride(0), k_cache.data_ptr(), vt_cache.data_ptr(), out.data_ptr(),
                                pos.data_ptr(), B, heads, kv_heads, D, L, Lc, cps, softmax_scale(scale, D), ws.ptr,
                                ws.bytes, stream_of(qkv)),
          "w4a8_attention_rope");
    return out;
}

// ------------------------------------------------------------------ 8-bit KV cache
struct Kv8 {
    int64_t B, KVH, NB, D;
    int code;
};

Kv8 check_kv8(const char* op, const Tensor& k_codes, const Tensor& vt_codes, const Tensor& kv_scale,
              const Tensor& k_tail, const Tensor& vt_tail, const Tensor& like) {
    const at::ScalarType dt = k_codes.scalar_type();
    TORCH_CHECK((dt == at::kChar || dt == at::kFloat8_e4m3fn) && vt_codes.scalar_type() == dt, op,
                ": codes must be int8 or float8_e4m3fn, K and V alike");
    TORCH_CHECK(k_codes.dim() == 5 && k_codes.size(1) > 0 && k_codes.size(2) > 0 && k_codes.size(3) == 64, op,
                ": k_codes must be [B, kv_heads, blocks, 64, head_dim], kv_heads and blocks > 0");
    const Kv8 s{k_codes.size(0), k_codes.size(1), k_codes.size(2), k_codes.size(4),
                dt == at::kChar ? W4A8_KV_INT8 : W4A8_KV_E4M3};
    TORCH_CHECK(vt_codes.sizes() == at::IntArrayRef({s.B, s.KVH, s.NB, s.D, 64}), op,
                ": vt_codes must be [B, kv_heads, blocks, head_dim, 64]");
    TORCH_CHECK(kv_scale.scalar_type() == at::kFloat && kv_scale.sizes() == at::IntArrayRef({s.B, s.KVH, s.NB, 2}), op,
                ": kv_scale must be float32 [B, kv_heads, blocks, 2]");
    TORCH_CHECK(k_tail.scalar_type() == at::kBFloat16 && k_tail.sizes() == at::IntArrayRef({s.B, s.KVH, 64, s.D}) &&
                    vt_tail.scalar_type() == at::kBFloat16 && vt_tail.sizes() == at::IntArrayRef({s.B, s.KVH, s.D, 64}),
                op, ": tails must be bfloat16 k [B, kv_heads, 64, head_dim] and vt [B, kv_heads, head_dim, 64]");
    for (const Tensor* t : {&k_codes, &vt_codes, &kv_scale, &k_tail, &vt_tail})
        TORCH_CHECK(t->is_contiguous() && t->device() == like.device(), op,
                    ": the cache must be contiguous and on one device with the other operands");
    return s;
}

// One position (length) for every sequence or one each; returns the stride between them.
int64_t check_pos(const char* op, const char* name, const Tensor& pos, int64_t B, const Tensor& like) {
    TORCH_CHECK(pos.scalar_type() == at::kLong && pos.dim() <= 1 && (pos.numel() == 1 || pos.numel() == B) &&
                    pos.device() == like.device(),
                op, ": ", name, " must be one int64 or one per sequence, on the device");
    return pos.numel() == 1 ? 0 : pos.stride(0);
}

void check_rope8(const char* op, const Tensor& cos, const Tensor& sin, int64_t L, int64_t D, const Tensor& like) {
    check_tables(op, cos, sin, L, D);
    TORCH_CHECK(cos.device() == like.device() && sin.device() == like.device(), op, ": cos and sin must be on the device");
}

// bf16 data that the kernels read sixteen bytes at a time.
Tensor aligned16(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 ? t.clone() : t; }

// The projection's output, B sequences of T rows of W (its strides st of sequence, row and
// element), with rows a distance `ld` apart that the kernels take: as it is or copied.  (The
// strides of dimensions of size one say nothing.)
Tensor projection(const Tensor& t, int64_t B, int64_t T, int64_t W, std::array<int64_t, 3> st, int64_t& ld) {
    ld = T > 1 ? st[1] : B > 1 ? st[0] : W;
    if (st[2] == 1 && ld >= W && ld % 8 == 0 && (B <= 1 || T <= 1 || st[0] == T * ld) &&
        reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0)
        return t;
    ld = W;
    return t.clone(at::MemoryFormat::Contiguous);
}

Tensor rope_kv8(const Tensor& qkv0, const Tensor& cos, const Tensor& sin, const Tensor& pos, const Tensor& k_codes,
                const Tensor& vt_codes, const Tensor& kv_scale, const Tensor& k_tail, const Tensor& vt_tail,
                int64_t heads, int64_t kv_heads, int64_t L, const std::optional<Tensor>& bias0) {
    TORCH_CHECK(qkv0.dim() == 3 && qkv0.scalar_type() == at::kBFloat16, "w4a8_rope_kv8: qkv must be bfloat16 [B, T, W]");
    const Kv8 c = check_kv8("w4a8_rope_kv8", k_codes, vt_codes, kv_scale, k_tail, vt_tail, qkv0);
    const int64_t B = qkv0.size(0), T = qkv0.size(1), W = qkv0.size(2);
    TORCH_CHECK(heads > 0 && kv_heads == c.KVH && B == c.B && W == (heads + 2 * kv_heads) * c.D,
                "w4a8_rope_kv8: qkv must be [B, T, (heads + 2 kv_heads) * head_dim] with the cache's B, kv_heads and "
                "head_dim");
    check_rope8("w4a8_rope_kv8", cos, sin, L, c.D, qkv0);
    const int64_t stride = check_pos("w4a8_rope_kv8", "pos", pos, B, qkv0);
    const at::DeviceGuard guard(qkv0.device());
    int64_t ld = 0;
    const Tensor qkv = projection(qkv0, B, T, W, {qkv0.stride(0), qkv0.stride(1), qkv0.stride(2)}, ld);
    auto bias = check_bias("w4a8_rope_kv8", bias0, W, qkv);
    if (bias.has_value()) bias = aligned16(*bias);
    Tensor q = empty({B, T, heads, c.D}, at::kBFloat16, qkv);
    check(abi().w4a8_rope_kv8(qkv.data_ptr(), ld, opt_ptr(bias), cos.data_ptr(), sin.data_ptr(),
                              cos.stride(0), pos.data_ptr(), stride, q.data_ptr(), k_codes.data_ptr(),
                              vt_codes.data_ptr(), kv_scale.data_ptr(), k_tail.data_ptr(), vt_tail.data_ptr(), c.code,
                              B, T, heads, kv_heads, c.D, L, c.NB, stream_of(qkv)),
          "w4a8_rope_kv8");
    return q;
}

std::tuple<Tensor, Tensor> kv8_read(const Tensor& k_codes, const Tensor& vt_codes, const Tensor& kv_scale,
                                    const Tensor& k_tail, const Tensor& vt_tail, const Tensor& length, int64_t first,
                                    int64_t n) {
    const Kv8 c = check_kv8("w4a8_kv8_read", k_codes, vt_codes, kv_scale, k_tail, vt_tail, k_codes);
    const int64_t stride = check_pos("w4a8_kv8_read", "length", length, c.B, k_codes);
    TORCH_CHECK(first >= 0 && n >= 0 && first <= 64 * c.NB && n <= 64 * c.NB - first, "w4a8_kv8_read: positions [",
                first, ", first + ", n, ") must lie inside the cache's ", 64 * c.NB);
    const at::DeviceGuard guard(k_codes.device());
    Tensor k = empty({c.B, c.KVH, n, c.D}, at::kBFloat16, k_codes), v = at::empty_like(k);
    check(abi().w4a8_kv8_read(k_codes.data_ptr(), vt_codes.data_ptr(), kv_scale.data_ptr(), k_tail.data_ptr(),
                              vt_tail.data_ptr(), c.code, length.data_ptr(), stride, k.data_ptr(), v.data_ptr(), first,
                              n, c.B, c.KVH, c.D, c.NB, stream_of(k_codes)),
          "w4a8_kv8_read");
    return {k, v};
}

Workspace kv8_workspace(const char* op, const Tensor& t, int64_t B, int64_t T, int64_t H, const Kv8& c, int64_t window,
                        int64_t sinks) {
    TORCH_CHECK(window >= 0 && sinks >= 0, op, ": window and sinks must be >= 0");
    const int64_t need = abi().w4a8_attention_kv8_workspace_bytes(B, T, H, c.KVH, c.D, c.NB, window, sinks);
    TORCH_CHECK(need >= 0, op, ": bad shape for the workspace size");
    return need > 0 ? workspace(t, need) : Workspace{};
}

Tensor attention_kv8(const Tensor& q0, const Tensor& k_codes, const Tensor& vt_codes, const Tensor& kv_scale,
                     const Tensor& k_tail, const Tensor& vt_tail, const Tensor& pos, int64_t L, int64_t window,
                     int64_t sinks, const std::optional<double>& scale) {
    TORCH_CHECK(q0.dim() == 4 && q0.scalar_type() == at::kBFloat16,
                "w4a8_attention_kv8: q must be bfloat16 [B, T, H, D]");
    const Kv8 c = check_kv8("w4a8_attention_kv8", k_codes, vt_codes, kv_scale, k_tail, vt_tail, q0);
    const int64_t B = q0.size(0), T = q0.size(1), H = q0.size(2);
    TORCH_CHECK(B == c.B && q0.size(3) == c.D && H % c.KVH == 0,
                "w4a8_attention_kv8: q must be [B, T, H, D] with the cache's B and D, H a multiple of its kv_heads");
    const int64_t stride = check_pos("w4a8_attention_kv8", "pos", pos, B, q0);
    const at::DeviceGuard guard(q0.device());
    const Tensor q = aligned16(q0.contiguous());
    Tensor out = empty({B, T, H, c.D}, at::kBFloat16, q);
    if (B * T == 0) return out;
    const Workspace ws = kv8_workspace("w4a8_attention_kv8", q, B, T, H, c, window, sinks);
    check(abi().w4a8_attention_kv8(q.data_ptr(), k_codes.data_ptr(), vt_codes.data_ptr(), kv_scale.data_ptr(),
                                   k_tail.data_ptr(), vt_tail.data_ptr(), c.code, out.data_ptr(), pos.data_ptr(),
                                   stride, B, T, H, c.KVH, c.D, L, c.NB, window, sinks, softmax_scale(scale, c.D),
                                   ws.ptr, ws.bytes, stream_of(q)),
          "w4a8_attention_kv8");
    return out;
}

Tensor attention_kv8_rope(const Tensor& qkv0, const Tensor& cos, const Tensor& sin, const Tensor& pos,
                          const Tensor& k_codes, const Tensor& vt_codes, const Tensor& kv_scale, const Tensor& k_tail,
                          const Tensor& vt_tail, int64_t heads, int64_t kv_heads, int64_t L,
                          const std::optional<Tensor>& bias0, int64_t window, int64_t sinks,
                          const std::optional<double>& scale) {
    TORCH_CHECK(qkv0.dim() == 2 && qkv0.scalar_type() == at::kBFloat16,
                "w4a8_attention_kv8_rope: qkv must be bfloat16 [B, W]");
    const Kv8 c = check_kv8("w4a8_attention_kv8_rope", k_codes, vt_codes, kv_scale, k_tail, vt_tail, qkv0);
    const int64_t B = qkv0.size(0), W = qkv0.size(1);
    TORCH_CHECK(heads > 0 && kv_heads == c.KVH && heads % kv_heads == 0 && B == c.B &&
                    W == (heads + 2 * kv_heads) * c.D,
                "w4a8_attention_kv8_rope: qkv must be [B, (heads + 2 kv_heads) * head_dim] with the cache's B, kv_heads "
                "and head_dim, heads a multiple of kv_heads");
    check_rope8("w4a8_attention_kv8_rope", cos, sin, L, c.D, qkv0);
    const int64_t stride = check_pos("w4a8_attention_kv8_rope", "pos", pos, B, qkv0);
    const at::DeviceGuard guard(qkv0.device());
    int64_t ld = 0;
    const Tensor qkv = projection(qkv0, B, 1, W, {qkv0.stride(0), W, qkv0.stride(1)}, ld);
    auto bias = check_bias("w4a8_attention_kv8_rope", bias0, W, qkv);
    if (bias.has_value()) bias = aligned16(*bias);
    Tensor out = empty({B, 1, heads, c.D}, at::kBFloat16, qkv);
    if (B == 0) return out;
    const Workspace ws = kv8_workspace("w4a8_attention_kv8_rope", qkv, B, 1, heads, c, window, sinks);
    check(abi().w4a8_attention_kv8_rope(qkv.data_ptr(), ld, opt_ptr(bias), cos.data_ptr(), sin.data_ptr(),
                                        cos.stride(0), k_codes.data_ptr(), vt_codes.data_ptr(), kv_scale.data_ptr(),
                                        k_tail.data_ptr(), vt_tail.data_ptr(), c.code, out.data_ptr(), pos.data_ptr(),
                                        stride, B, heads, kv_heads, c.D, L, c.NB, window, sinks,
                                        softmax_scale(scale, c.D), ws.ptr, ws.bytes, stream_of(qkv)),
          "w4a8_attention_kv8_rope");
    return out;
}

// ------------------------------------------------------------------ mid-group compat pair
int64_t padded_rows(int64_t M) {
    const int64_t t = M <= 16 ? 16 : (M <= 64 ? 64 : 128);
    return geom::ceil_to(M, t);
}

std::vector<Tensor> midgroup_quant_a(const Tensor& x0, int64_t group) {
    TORCH_CHECK(x0.dim() == 2, "midgroup_quant_a: x must be [M, K]");
    TORCH_CHECK(x0.scalar_type() == at::kBFloat16, "midgroup_quant_a: x must be bfloat16");
    TORCH_CHECK(group > 0, "midgroup_quant_a: group must be > 0");
    const Tensor x = rows(x0);
    const int64_t M = x.size(0), K = x.size(1);
    check_geometry("midgroup_quant_a", K, group);
    const int64_t G = geom::num_groups(K, group), kb = geom::kpad(K, group) / 2, Mp = M ? padded_rows(M) : 0;
    Tensor a_hi = empty({Mp, kb}, at::kChar, x), a_lo = empty({Mp, kb}, at::kChar, x);
    Tensor a_scale = empty({G, Mp}, at::kBFloat16, x), a_ksum = empty({G, Mp}, at::kInt, x);
    if (Mp)
        check(abi().w4a8_midgroup_quant_a(x.data_ptr(), x.stride(0), a_hi.data_ptr(), a_lo.data_ptr(),
                                          a_scale.data_ptr(), a_ksum.data_ptr(), M, Mp, K, group, stream_of(x)),
              "midgroup_quant_a");
    return {a_hi, a_lo, a_scale, a_ksum};
}

// w_q is [N, kpad/2], or with tiled the midgroup_tile_weights tiles of such a weight.
Tensor run_midgroup(const Tensor& a_hi0, const Tensor& a_lo0, const Tensor& a_scale0, const Tensor& a_ksum0,
                    const Tensor& w_q0, const Tensor& w_scale0, const Tensor& w_ksum, const Tensor& w_zero0, int64_t N,
                    int64_t K, int64_t group, int64_t nrows, bool tiled) {
    check_geometry("midgroup_w4a8_gemm", K, group);
    const Abi& f = abi();
    const int64_t kb = geom::kpad(K, group) / 2, G = geom::num_groups(K, group);
    if (tiled) {
        const int64_t nbytes = f.w4a8_midgroup_tiles_bytes(N, K, group);
        TORCH_CHECK(w_q0.scalar_type() == at::kChar && w_q0.numel() == nbytes && w_q0.is_contiguous(),
                    "midgroup_w4a8_gemm_tiled: w_tiles must be the ", nbytes, " int8 bytes of midgroup_tile_weights");
    }
    TORCH_CHECK(a_hi0.dim() == 2 && a_lo0.dim() == 2 && (tiled || w_q0.dim() == 2),
                "midgroup_w4a8_gemm: a_hi/a_lo [M,K/2] and w_q [N,K/2] must be 2-D");
    TORCH_CHECK(a_hi0.scalar_type() == at::kChar && a_lo0.scalar_type() == at::kChar && w_q0.scalar_type() == at::kChar,
                "midgroup_w4a8_gemm: packed int4 planes must be int8 tensors");
    TORCH_CHECK(a_scale0.scalar_type() == at::kBFloat16 && w_scale0.scalar_type() == at::kBFloat16 &&
                    w_zero0.scalar_type() == at::kBFloat16,
                "midgroup_w4a8_gemm: a_scale/w_scale/w_zero must be bfloat16");
    TORCH_CHECK(a_ksum0.scalar_type() == at::kInt && w_ksum.scalar_type() == at::kInt,
                "midgroup_w4a8_gemm: a_ksum/w_ksum must be int32");
    TORCH_CHECK(a_hi0.size(1) == kb && a_lo0.sizes() == a_hi0.sizes() && (tiled || w_q0.size(1) == kb),
                "midgroup_w4a8_gemm: packed row length must be Kpad/2 = ", kb, " for K=", K,
                " (group-padded layout); got a_hi ", a_hi0.size(1), " w_q ", tiled ? kb : w_q0.size(1));
    int64_t M = a_hi0.size(0);
    if (!tiled) N = w_q0.size(0);
    TORCH_CHECK(a_scale0.dim() == 2 && a_scale0.size(0) == G && a_scale0.size(1) >= M &&
                    a_ksum0.sizes() == a_scale0.sizes(),
                "midgroup_w4a8_gemm: a_scale/a_ksum must be group-major [K/group, M]");
    const int64_t gn[2] = {G, N};
    TORCH_CHECK(w_scale0.sizes() == at::IntArrayRef(gn, 2) && w_zero0.sizes() == at::IntArrayRef(gn, 2) &&
                    w_ksum.sizes() == at::IntArrayRef(gn, 2),
                "midgroup_w4a8_gemm: w_scale/w_zero/w_ksum must be group-major [K/group, N]");
    if (nrows >= 0) {
        // the first rows only (the real rows before quant_a's padding): the padding
        // rows' activation planes are then never read
        TORCH_CHECK(nrows <= M, "midgroup_w4a8_gemm: rows=", nrows, " exceeds the ", M, " activation rows");
        M = nrows;
    }
    const Tensor a_hi = a_hi0.contiguous(), a_lo = a_lo0.contiguous(), w_q = w_q0.contiguous();
    const Tensor a_scale = a_scale0.contiguous(), a_ksum = a_ksum0.contiguous();
    const Tensor w_scale = w_scale0.contiguous(), w_zero = w_zero0.contiguous();
    Tensor y = empty({M, N}, at::kBFloat16, a_hi);
    if (M == 0) return y;
    // w_ksum is validated but not read: the activation bytes are rebuilt exactly from
    // the two planes, so the kernel needs no +8 correction.  Few rows on a long K get a
    // workspace for the int32 group sums of a split K, prefill sizes one for the rebuilt
    // rows, allocated per call as the reference host allocates its GEMM workspace
    // (npu_ops/host/midgroup_w4a8_gemm.cpp:116-118).
    Tensor ws;
    if (const int64_t sums = f.w4a8_midgroup_split_workspace_bytes(M, N, K, group)) {
        ws = empty({sums}, at::kByte, a_hi);
        check(f.w4a8_midgroup_gemm_split(a_hi.data_ptr(), a_lo.data_ptr(), a_scale.data_ptr(), a_ksum.data_ptr(), M,
                                         a_scale.stride(0), w_q.data_ptr(), tiled, w_scale.data_ptr(),
                                         w_zero.data_ptr(), y.data_ptr(), N, N, K, group, ws.data_ptr(), sums,
                                         stream_of(a_hi)),
              "midgroup_w4a8_gemm");
        return y;
    }
    const int64_t need = f.w4a8_midgroup_gemm_workspace_bytes(M, N, K, group);
    if (need) ws = empty({need}, at::kByte, a_hi);
    check((tiled ? f.w4a8_midgroup_gemm_tiled : f.w4a8_midgroup_gemm_ws)(
              a_hi.data_ptr(), a_lo.data_ptr(), a_scale.data_ptr(), a_ksum.data_ptr(), M, a_scale.stride(0),
              w_q.data_ptr(), w_scale.data_ptr(), w_zero.data_ptr(), y.data_ptr(), N, nullptr, N, K, group,
              need ? ws.data_ptr() : nullptr, need, stream_of(a_hi)),
          "midgroup_w4a8_gemm");
    return y;
}

Tensor midgroup_gemm(const Tensor& a_hi, const Tensor& a_lo, const Tensor& a_scale, const Tensor& a_ksum,
                     const Tensor& w_q, const Tensor& w_scale, const Tensor& w_ksum, const Tensor& w_zero, int64_t K,
                     int64_t group, int64_t nrows) {
    return run_midgroup(a_hi, a_lo, a_scale, a_ksum, w_q, w_scale, w_ksum, w_zero, -1, K, group, nrows, false);
}

Tensor midgroup_gemm_tiled(const Tensor& a_hi, const Tensor& a_lo, const Tensor& a_scale, const Tensor& a_ksum,
                           const Tensor& w_tiles, const Tensor& w_scale, const Tensor& w_ksum, const Tensor& w_zero,
                           int64_t N, int64_t K, int64_t group, int64_t nrows) {
    return run_midgroup(a_hi, a_lo, a_scale, a_ksum, w_tiles, w_scale, w_ksum, w_zero, N, K, group, nrows, true);
}

TORCH_LIBRARY_IMPL(npu, CUDA, m) {
    m.impl("w4a8_quant_pertoken", &quant_pertoken);
    m.impl("w4a8_gemm", &gemm);
    m.impl("w4a8_gemm_swiglu", &gemm_swiglu);
    m.impl("w4a8_linear", &linear);
    m.impl("w4a8_rmsnorm_quant", &rmsnorm_quant);
    m.impl("w4a8_rope_kv", &rope_kv);
    m.impl("w4a8_attention", &attention);
    m.impl("w4a8_attention_rope", &attention_rope);
    m.impl("w4a8_rope_kv8", &rope_kv8);
    m.impl("w4a8_kv8_read", &kv8_read);
    m.impl("w4a8_attention_kv8", &attention_kv8);
    m.impl("w4a8_attention_kv8_rope", &attention_kv8_rope);
    m.impl("midgroup_quant_a", &midgroup_quant_a);
    m.impl("midgroup_w4a8_gemm", &midgroup_gemm);
    m.impl("midgroup_w4a8_gemm_tiled", &midgroup_gemm_tiled);
}

}  // namespace

PYBIND11_MODULE(w4a8_torch, m) {
    m.def("abi_names", &abi_names);
    m.def("init", [](py::object loader, py::object ws) {
        g_loader = loader.release().ptr();
        g_workspace = ws.release().ptr();
    });
}
