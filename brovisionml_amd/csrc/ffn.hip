// The C ABI of the feed-forward operators (include/bvml_ffn.h): every check of
// arguments, then the launches.  Nothing here allocates or synchronises.

#include <cmath>
#include <cstring>
#include <initializer_list>
#include <new>
#include <string>

#include "bvml_ffn.h"
#include "ffn_kernels.h"
#include "status.h"

namespace {

using bvml::fail;
using namespace bvml_ffn;

constexpr int kMostNormCols = 32768;
// A tile's offsets are 32-bit byte offsets from its first row: 256 rows of at
// most this many bytes.
constexpr long long kMostRowBytes = (1LL << 31) / 256 - 256;
constexpr long long kMostRows = (1LL << 31) - 512;

int size_of(int type) { return type == kF32 ? 4 : type == kE4M3 ? 1 : 2; }
bool is16(int type) { return type == kF16 || type == kBF16; }
bool is_value(int type) { return type == kF32 || is16(type); }

// An array argument: rows x cols elements of `type`, rows ld elements apart.
struct Array {
    const char* name;
    const void* p;
    long long ld;
    long long rows, cols;
    int type;
    size_t bytes() const {
        return rows > 0 ? ((size_t)(rows - 1) * ld + cols) * size_of(type) : 0;
    }
};

int check_array(const std::string& op, const Array& a, bool optional) {
    if (a.p == nullptr) {
        if (optional || a.rows == 0) return BVML_FFN_OK;
        return fail(BVML_FFN_ENULL, op + ": " + a.name + " is NULL");
    }
    if (a.ld < a.cols)
        return fail(BVML_FFN_ESHAPE, op + ": rows of " + a.name + " are closer than their width");
    if (a.ld * size_of(a.type) > kMostRowBytes)
        return fail(BVML_FFN_ESIZE, op + ": rows of " + a.name + " are too far apart");
    return BVML_FFN_OK;
}

// No output may overlap an input or another output, but `may_out` may be any of
// `may_in` itself, element for element.
int check_alias(const std::string& op, std::initializer_list<Array> outs,
                std::initializer_list<Array> ins, const char* may_out,
                std::initializer_list<const char*> may_in) {
    const Array* o = outs.begin();
    for (size_t i = 0; i < outs.size(); ++i) {
        if (o[i].p == nullptr || o[i].bytes() == 0) continue;
        for (size_t j = i + 1; j < outs.size(); ++j)
            if (o[j].p && bvml::overlaps(o[i].p, o[i].bytes(), o[j].p, o[j].bytes()))
                return fail(BVML_FFN_EALIAS, op + ": " + o[i].name + " overlaps " + o[j].name);
        for (const Array& in : ins) {
            if (!in.p || !bvml::overlaps(o[i].p, o[i].bytes(), in.p, in.bytes())) continue;
            bool may = false;
            if (may_out && std::strcmp(may_out, o[i].name) == 0 && in.p == o[i].p &&
                in.ld == o[i].ld && in.type == o[i].type)
                for (const char* name : may_in) may = may || std::strcmp(name, in.name) == 0;
            if (!may) return fail(BVML_FFN_EALIAS, op + ": " + o[i].name + " overlaps " + in.name);
        }
    }
    return BVML_FFN_OK;
}

#define BVML_FFN_TRY(x)                    \
    do {                                   \
        const int status_ = (x);           \
        if (status_ != BVML_FFN_OK) return status_; \
    } while (0)

int launched(const std::string& op, hipError_t e) {
    if (e == hipSuccess) return BVML_FFN_OK;
    if (e == hipErrorInvalidConfiguration)
        return fail(BVML_FFN_ESIZE, op + ": more tiles than a launch holds");
    return fail((int)e, op + ": " + hipGetErrorString(e));
}

// An entry point's body: nothing is thrown past it.  (What can be thrown is that
// a message's memory is not there; the last message then stays.)
template <typename F>
int guarded(F body) noexcept {
    try {
        return body();
    } catch (const std::bad_alloc&) {
        return (int)hipErrorOutOfMemory;
    }
}

int check_act(const std::string& op, int act) {
    if (act < BVML_FFN_NONE || act > BVML_FFN_SILU)
        return fail(BVML_FFN_EPARAM, op + ": unknown activation");
    return BVML_FFN_OK;
}

int check_sizes(const std::string& op, int M, int N, int K, bool gated) {
    if (M < 0 || N < 1 || K < 1)
        return fail(BVML_FFN_ESHAPE, op + ": M must be >= 0, N and K >= 1");
    if (M > kMostRows || (long long)N * (gated ? 2 : 1) > kMostRows)
        return fail(BVML_FFN_ESIZE, op + ": too many rows");
    return BVML_FFN_OK;
}

long long round256(long long n) { return (n + 255) / 256 * 256; }

// linear and gated
int forward(const std::string& op, bool gated, const void* x, long long ldx, const void* w,
            long long ldw, const void* bias, const float* x_scale, const float* w_scale,
            const void* residual, long long ldr, int M, int N, int K, int in_type, int out_type,
            int bias_type, int act, void* y, long long ldy, void* z, long long ldz,
            void* workspace, long long workspace_bytes, void* stream) {
    BVML_FFN_TRY(check_sizes(op, M, N, K, gated));
    BVML_FFN_TRY(check_act(op, act));
    const bool e4m3 = in_type == kE4M3;
    if (!e4m3 && !is16(in_type))
        return fail(BVML_FFN_ETYPE, op + ": x and w must be f16, bf16 or e4m3");
    if (!is_value(out_type) || (!e4m3 && out_type != kF32 && out_type != in_type))
        return fail(BVML_FFN_ETYPE, op + ": the output is of x's 16-bit type or f32 (from e4m3: "
                                         "f16, bf16 or f32)");
    if (bias && bias_type != kF32 && bias_type != out_type && (e4m3 || bias_type != in_type))
        return fail(BVML_FFN_ETYPE, op + ": the bias is f32 or of the output's or x's type");
    if (e4m3 != (x_scale != nullptr) || e4m3 != (w_scale != nullptr))
        return fail(e4m3 ? BVML_FFN_ENULL : BVML_FFN_ETYPE,
                    op + ": e4m3 operands, and no others, come with x_scale and w_scale");
    if (z && e4m3)
        return fail(BVML_FFN_ETYPE, op + ": pre-activations are kept for 16-bit operands only");
    const long long R = gated ? 2LL * N : N;
    const Array ax{"x", x, ldx, M, K, in_type}, aw{"w", w, ldw, R, K, in_type};
    const Array ar{"residual", residual, ldr, M, N, out_type};
    const Array ay{gated ? "h" : "y", y, ldy, M, N, out_type}, az{"z", z, ldz, M, R, in_type};
    const Array ab{"bias", bias, R, 1, R, bias_type};
    const Array axs{"x_scale", x_scale, M, 1, M, kF32}, aws{"w_scale", w_scale, R, 1, R, kF32};
    BVML_FFN_TRY(check_array(op, ax, false));
    BVML_FFN_TRY(check_array(op, aw, M == 0));
    BVML_FFN_TRY(check_array(op, ar, true));
    BVML_FFN_TRY(check_array(op, ay, false));
    BVML_FFN_TRY(check_array(op, az, true));
    BVML_FFN_TRY(check_alias(op, {ay, az}, {ax, aw, ar, ab, axs, aws}, "y", {"residual"}));
    if (M == 0) return BVML_FFN_OK;
    const long long need = product_workspace(M, (int)R, K, in_type, kForward, gated);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need))
        return fail(BVML_FFN_EWORK, op + ": the workspace must hold " + std::to_string(need) +
                                        " bytes");
    if (need > 0) {
        const Array awork{"the workspace", workspace, need, 1, need, kE4M3};
        BVML_FFN_TRY(check_alias(op, {awork}, {ax, aw, ar, ab, axs, aws, ay, az}, nullptr, {}));
        if (((uintptr_t)workspace & 15) != 0)
            return fail(BVML_FFN_EWORK, op + ": the workspace must begin on 16 bytes");
    }
    ProductCall c{};
    c.p = x;
    c.q = w;
    c.ldp = ldx;
    c.ldq = ldw;
    c.M = M;
    c.R = (int)R;
    c.K = K;
    c.in_type = in_type;
    c.layout = kForward;
    c.gated = gated;
    c.padded_p = false;
    c.e = Epilogue{bias, x_scale, w_scale, residual, y, z, nullptr, ldr, ldy, ldz, M, N,
                   bias_type, out_type, in_type, act};
    return launched(op, launch_product(c, workspace, static_cast<hipStream_t>(stream)));
}

// The workspace of a backward pass, in order: dz, the slope's partial sums,
// a split product's.
struct GradSpace {
    long long dz, sums, parts;
    GradSpace(int M, int R, int K, int type) {
        const long long ldd = (R + 7LL) / 8 * 8;
        dz = round256(M * ldd * 2);
        sums = round256(slope_workspace(M, R));
        const long long a = product_workspace(M, K, R, type, kInputGrad, false);
        const long long b = product_workspace(R, K, M, type, kWeightGrad, false);
        const long long c = gradients_workspace(M, R, K);
        parts = a > b ? a : b;
        if (c > parts) parts = c;
    }
    long long all() const { return dz + sums + parts; }
};

int backward(const std::string& op, bool gated, const void* dy, long long lddy, const void* x,
             long long ldx, const void* w, long long ldw, const void* z, long long ldz, int M,
             int N, int K, int type, int dy_type, int act, void* dx, long long lddx, void* dw,
             long long lddw, void* db, void* workspace, long long workspace_bytes, void* stream) {
    BVML_FFN_TRY(check_sizes(op, M, N, K, gated));
    BVML_FFN_TRY(check_act(op, act));
    if (!is16(type)) return fail(BVML_FFN_ETYPE, op + ": x and w must be f16 or bf16");
    if (dy_type != type && dy_type != kF32)
        return fail(BVML_FFN_ETYPE, op + ": the output's gradient must be f32 or of x's type");
    const int R = gated ? 2 * N : N;
    const bool sloped = gated || act != BVML_FFN_NONE;
    const Array ady{gated ? "dh" : "dy", dy, lddy, M, N, dy_type};
    const Array ax{"x", x, ldx, M, K, type}, aw{"w", w, ldw, R, K, type};
    const Array az{"z", z, ldz, M, R, type};
    const Array adx{"dx", dx, lddx, M, K, type}, adw{"dw", dw, lddw, R, K, type};
    const Array adb{"db", db, R, 1, R, type};
    BVML_FFN_TRY(check_array(op, ady, false));
    BVML_FFN_TRY(check_array(op, ax, dw == nullptr));
    BVML_FFN_TRY(check_array(op, aw, dx == nullptr || M == 0));
    BVML_FFN_TRY(check_array(op, az, !sloped));
    BVML_FFN_TRY(check_array(op, adx, true));
    BVML_FFN_TRY(check_array(op, adw, true));
    BVML_FFN_TRY(check_alias(op, {adx, adw, adb}, {ady, ax, aw, az}, nullptr, {}));
    if (!dx && !dw && !db) return BVML_FFN_OK;
    const GradSpace space(M, R, K, type);
    if (space.all() > 0 && (workspace == nullptr || workspace_bytes < space.all()))
        return fail(BVML_FFN_EWORK, op + ": the workspace must hold " +
                                        std::to_string(space.all()) + " bytes");
    const Array awork{"the workspace", workspace, space.all(), 1, space.all(), kE4M3};
    BVML_FFN_TRY(check_alias(op, {awork}, {ady, ax, aw, az, adx, adw, adb}, nullptr, {}));
    if (((uintptr_t)workspace & 15) != 0)
        return fail(BVML_FFN_EWORK, op + ": the workspace must begin on 16 bytes");
    hipStream_t s = static_cast<hipStream_t>(stream);
    char* const at = static_cast<char*>(workspace);

    SlopeCall sc{};
    sc.dy = dy;
    sc.z = sloped ? z : nullptr;
    sc.lddy = lddy;
    sc.ldz = ldz;
    sc.ldd = (R + 7LL) / 8 * 8;
    sc.rows = M;
    sc.N = N;
    sc.gated = gated;
    sc.dy_type = dy_type;
    sc.type = type;
    sc.act = act;
    // without an activation dz is dy, already in the products' type
    const bool own_dz = sloped || dy_type != type;
    sc.dz = own_dz && (dx || dw) ? at : nullptr;
    sc.db = db;
    sc.workspace = reinterpret_cast<float*>(at + space.dz);
    ColumnSum sums{};
    if (sc.dz || sc.db) BVML_FFN_TRY(launched(op, launch_slope(sc, &sums, s)));

    ProductCall c{};
    c.p = own_dz ? at : dy;
    c.ldp = own_dz ? sc.ldd : lddy;
    c.in_type = type;
    c.gated = false;
    c.padded_p = own_dz;
    auto plain = [&](void* y, long long ldy, int rows) {
        return Epilogue{nullptr, nullptr, nullptr, nullptr, y, nullptr, nullptr, 0, ldy, 0, rows, K,
                        type, type, type, BVML_FFN_NONE};
    };
    ProductCall input = c, weight = c;
    input.q = w;
    input.ldq = ldw;
    input.M = M;
    input.R = K;
    input.K = R;
    input.layout = kInputGrad;
    input.e = plain(dx, lddx, M);
    weight.q = x;
    weight.ldq = ldx;
    weight.M = R;
    weight.R = K;
    weight.K = M;
    weight.layout = kWeightGrad;
    weight.e = plain(dw, lddw, R);
    void* const parts = at + space.dz + space.sums;
    if (dx && dw) return launched(op, launch_gradients(input, weight, sums, parts, s));
    if (db) BVML_FFN_TRY(launched(op, launch_column_sum(sums, s)));
    if (dx && M > 0) return launched(op, launch_product(input, parts, s));
    if (dw) return launched(op, launch_product(weight, parts, s));
    return BVML_FFN_OK;
}

}  // namespace

extern "C" {

int bvml_ffn_add_rms_norm(const void* x, long long ldx, const void* residual, long long ldr,
                          const void* weight, int rows, int cols, double eps, int x_type,
                          int w_type, int y_type, void* y, long long ldy, void* stream_out,
                          long long lds, float* scale, float* rstd, void* stream) {
    return guarded([&]() -> int {
        const std::string op = "add_rms_norm";
        if (rows < 0 || cols < 1)
            return fail(BVML_FFN_ESHAPE, op + ": rows must be >= 0, cols >= 1");
        if (cols > kMostNormCols) return fail(BVML_FFN_ESIZE, op + ": more than 32768 columns");
        if (rows > kMostRows) return fail(BVML_FFN_ESIZE, op + ": too many rows");
        if (!(eps >= 0.0) || !std::isfinite((float)eps))
            return fail(BVML_FFN_EPARAM, op + ": eps must be >= 0 and finite in fp32");
        if (!is_value(x_type)) return fail(BVML_FFN_ETYPE, op + ": x must be f32, f16 or bf16");
        if (weight && w_type != kF32 && w_type != x_type)
            return fail(BVML_FFN_ETYPE, op + ": the weight must be f32 or of x's type");
        if (y_type != x_type && y_type != kE4M3 && !(x_type == kF32 && is16(y_type)))
            return fail(BVML_FFN_ETYPE,
                        op + ": y must be of x's type, e4m3, or (from f32) 16 bits");
        if ((y_type == kE4M3) != (scale != nullptr) && !(rows == 0 && scale == nullptr))
            return fail(scale ? BVML_FFN_ETYPE : BVML_FFN_ENULL,
                        op + ": e4m3 output, and no other, comes with scale");
        const Array ax{"x", x, ldx, rows, cols, x_type};
        const Array ar{"residual", residual, ldr, rows, cols, x_type};
        const Array aw{"weight", weight, cols, 1, cols, w_type};
        const Array ay{"y", y, ldy, rows, cols, y_type};
        const Array as{"stream", stream_out, lds, rows, cols, x_type};
        const Array ac{"scale", scale, rows, 1, rows, kF32}, ad{"rstd", rstd, rows, 1, rows, kF32};
        BVML_FFN_TRY(check_array(op, ax, false));
        BVML_FFN_TRY(check_array(op, ar, true));
        BVML_FFN_TRY(check_array(op, ay, false));
        BVML_FFN_TRY(check_array(op, as, true));
        BVML_FFN_TRY(check_alias(op, {ay, as, ac, ad}, {ax, ar, aw}, "stream", {"x", "residual"}));
        if (rows == 0) return BVML_FFN_OK;
        const NormCall c{x, residual, weight, ldx, ldr, ldy, lds, rows, cols, (float)eps, x_type,
                         w_type, y_type, y, stream_out, scale, rstd};
        return launched(op, launch_norm(c, static_cast<hipStream_t>(stream)));
    });
}

long long bvml_ffn_add_rms_norm_backward_workspace(int rows, int cols) {
    return rows < 0 || cols < 1 || cols > kMostNormCols ? -1 : norm_grad_workspace(rows, cols);
}

int bvml_ffn_add_rms_norm_backward(const void* dy, long long lddy, const void* s, long long lds,
                                   const void* weight, const float* rstd, const void* dstream,
                                   long long lddst, int rows, int cols, int dy_type, int s_type,
                                   int w_type, void* ds, long long ldds, void* dweight,
                                   void* workspace, long long workspace_bytes, void* stream) {
    return guarded([&]() -> int {
        const std::string op = "add_rms_norm_backward";
        if (rows < 0 || cols < 1)
            return fail(BVML_FFN_ESHAPE, op + ": rows must be >= 0, cols >= 1");
        if (cols > kMostNormCols) return fail(BVML_FFN_ESIZE, op + ": more than 32768 columns");
        if (rows > kMostRows) return fail(BVML_FFN_ESIZE, op + ": too many rows");
        if (!is_value(s_type) || !is_value(dy_type))
            return fail(BVML_FFN_ETYPE, op + ": s and dy must be f32, f16 or bf16");
        if ((weight || dweight) && w_type != kF32 && w_type != s_type)
            return fail(BVML_FFN_ETYPE, op + ": the weight must be f32 or of s's type");
        const Array ady{"dy", dy, lddy, rows, cols, dy_type}, as{"s", s, lds, rows, cols, s_type};
        const Array aw{"weight", weight, cols, 1, cols, w_type};
        const Array ar{"rstd", rstd, rows, 1, rows, kF32};
        const Array adst{"dstream", dstream, lddst, rows, cols, s_type};
        const Array ads{"ds", ds, ldds, rows, cols, s_type};
        const Array adw{"dweight", dweight, cols, 1, cols, w_type};
        BVML_FFN_TRY(check_array(op, ady, false));
        BVML_FFN_TRY(check_array(op, as, false));
        if (rows > 0 && rstd == nullptr) return fail(BVML_FFN_ENULL, op + ": rstd is NULL");
        BVML_FFN_TRY(check_array(op, adst, true));
        BVML_FFN_TRY(check_array(op, ads, false));
        BVML_FFN_TRY(check_alias(op, {ads, adw}, {ady, as, aw, ar, adst}, "ds", {"dstream"}));
        const long long need = dweight ? norm_grad_workspace(rows, cols) : 0;
        if (need > 0 && (workspace == nullptr || workspace_bytes < need))
            return fail(BVML_FFN_EWORK, op + ": the workspace must hold " + std::to_string(need) +
                                            " bytes");
        const Array awork{"the workspace", workspace, need, need > 0, need, kE4M3};
        BVML_FFN_TRY(check_alias(op, {awork}, {ady, as, aw, ar, adst, ads, adw}, nullptr, {}));
        const NormGradCall c{dy, s, weight, rstd, dstream, lddy, lds, lddst, ldds, rows, cols,
                             dy_type, s_type, w_type, ds, dweight, static_cast<float*>(workspace)};
        return launched(op, launch_norm_grad(c, static_cast<hipStream_t>(stream)));
    });
}

int bvml_ffn_linear(const void* x, long long ldx, const void* w, long long ldw, const void* bias,
                    const float* x_scale, const float* w_scale, const void* residual,
                    long long ldr, int M, int N, int K, int in_type, int out_type, int bias_type,
                    int act, void* y, long long ldy, void* z, long long ldz, void* workspace,
                    long long workspace_bytes, void* stream) {
    return guarded([&]() -> int {
        return forward("linear", false, x, ldx, w, ldw, bias, x_scale, w_scale, residual, ldr, M,
                       N, K, in_type, out_type, bias_type, act, y, ldy, z, ldz, workspace,
                       workspace_bytes, stream);
    });
}

long long bvml_ffn_linear_workspace(int M, int N, int K, int in_type) {
    if (M < 0 || N < 1 || K < 1) return -1;
    return product_workspace(M, N, K, in_type, kForward, false);
}

int bvml_ffn_gated(const void* x, long long ldx, const void* w, long long ldw, const void* bias,
                   const float* x_scale, const float* w_scale, int M, int N, int K, int in_type,
                   int out_type, int bias_type, int act, void* h, long long ldh, void* z,
                   long long ldz, void* workspace, long long workspace_bytes, void* stream) {
    return guarded([&]() -> int {
        return forward("gated", true, x, ldx, w, ldw, bias, x_scale, w_scale, nullptr, 0, M, N, K,
                       in_type, out_type, bias_type, act, h, ldh, z, ldz, workspace,
                       workspace_bytes, stream);
    });
}

long long bvml_ffn_gated_workspace(int M, int N, int K, int in_type) {
    if (M < 0 || N < 1 || N > kMostRows / 2 || K < 1) return -1;
    return product_workspace(M, 2 * N, K, in_type, kForward, true);
}

int bvml_ffn_linear_backward(const void* dy, long long lddy, const void* x, long long ldx,
                             const void* w, long long ldw, const void* z, long long ldz, int M,
                             int N, int K, int type, int dy_type, int act, void* dx,
                             long long lddx, void* dw, long long lddw, void* db, void* workspace,
                             long long workspace_bytes, void* stream) {
    return guarded([&]() -> int {
        return backward("linear_backward", false, dy, lddy, x, ldx, w, ldw, z, ldz, M, N, K, type,
                        dy_type, act, dx, lddx, dw, lddw, db, workspace, workspace_bytes, stream);
    });
}

long long bvml_ffn_linear_backward_workspace(int M, int N, int K) {
    if (M < 0 || N < 1 || K < 1) return -1;
    return GradSpace(M, N, K, kBF16).all();
}

int bvml_ffn_gated_backward(const void* dh, long long lddh, const void* x, long long ldx,
                            const void* w, long long ldw, const void* z, long long ldz, int M,
                            int N, int K, int type, int dh_type, int act, void* dx,
                            long long lddx, void* dw, long long lddw, void* db, void* workspace,
                            long long workspace_bytes, void* stream) {
    return guarded([&]() -> int {
        return backward("gated_backward", true, dh, lddh, x, ldx, w, ldw, z, ldz, M, N, K, type,
                        dh_type, act, dx, lddx, dw, lddw, db, workspace, workspace_bytes, stream);
    });
}

long long bvml_ffn_gated_backward_workspace(int M, int N, int K) {
    if (M < 0 || N < 1 || N > kMostRows / 2 || K < 1) return -1;
    return GradSpace(M, 2 * N, K, kBF16).all();
}

int bvml_ffn_plan(int M, int R, int K, int in_type, int layout, int gated, int aligned, int* tile,
                  int* deep, int* whole, int* splits) {
    return guarded([&]() -> int {
        if (M < 1 || R < 1 || K < 1)
            return fail(BVML_FFN_ESHAPE, "plan: sizes must be >= 1");
        if ((in_type != kE4M3 && !is16(in_type)) || layout < kForward || layout > kWeightGrad + 1 ||
            (layout != kForward && (gated || in_type == kE4M3)))
            return fail(BVML_FFN_ETYPE, "plan: no such product");
        ProductPlan p;
        if (layout <= kWeightGrad) {
            p = plan_product(M, R, K, in_type, layout, gated != 0, aligned != 0);
        } else {
            const GradientsPlan g = plan_gradients(M, R, K);
            p = {g.tile, true, g.input_splits > 1 ? g.input_whole : g.weight_whole,
                 g.input_splits > 1 ? g.input_splits : g.weight_splits};
        }
        static const int kRows[] = {256, 128, 128, 64, 64, 0};  // by Tile
        if (tile) *tile = kRows[p.tile];
        if (deep) *deep = p.tile == kTile128Deep || p.tile == kTileSquare;
        if (whole) *whole = p.whole;
        if (splits) *splits = p.splits;
        return BVML_FFN_OK;
    });
}

const char* bvml_ffn_last_error(void) { return bvml::last_error(); }

const char* bvml_ffn_version(void) { return "0.1.0"; }

}  // extern "C"
