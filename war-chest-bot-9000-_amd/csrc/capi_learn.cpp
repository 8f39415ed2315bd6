// The training operators' entry points (include/wc_learn.h): every argument is
// checked here, before anything is queued.
#include <exception>
#include <mutex>
#include <string>

#include "../../include/wc_learn.h"
#include "common.h"
#include "learn.h"

using namespace wc;

namespace {

constexpr int64_t MOST = int64_t(1) << 40;     // rows, widths and strides beyond any memory
constexpr int64_t MOST_LANES = int64_t(1) << 31;  // widths and pairs that index a grid

// The checks of one call: the first that fails is the one told.
struct Check {
    const char* what;
    int code = WC_OK;
    std::string msg;

    bool is(bool ok, const char* text, int c = WC_ERR_INVALID) {
        if (!ok && code == WC_OK) {
            code = c;
            msg = std::string(what) + ": " + text;
        }
        return ok;
    }
    bool aligned(const void* p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }
    // A buffer that must be there if `rows` is not 0, of elements of n bytes.
    void buffer(const void* p, size_t n, bool need, const char* name) {
        if (need && !p) is(false, (std::string(name) + " is missing").c_str());
        if (p && !aligned(p, n)) is(false, (std::string(name) + " is not aligned to its elements").c_str());
    }
    void matrix(const void* p, size_t n, int64_t stride, int64_t width, int64_t rows, bool written, bool need,
                const char* name) {
        buffer(p, n, need, name);
        if (!p) return;
        if (stride < 0 || stride > MOST || (written && rows > 1 && stride < width) || (stride && rows > 1 && stride < width))
            is(false, (std::string(name) + ": rows overlap or the stride is out of range").c_str());
    }
    // An output that may be an input itself lies as that does: its rows are read where they are written, and by no one else.
    void over(const void* out, int64_t out_stride, const void* in, int64_t in_stride, int64_t rows, const char* names) {
        if (out && out == in && rows > 1 && out_stride != in_stride)
            is(false, (std::string(names) + " itself needs its row stride").c_str());
    }
};

size_t size_of(int dtype) { return dtype == WC_DTYPE_F32 ? 4 : 2; }

bool known(int dtype) { return dtype == WC_DTYPE_F32 || dtype == WC_DTYPE_F16 || dtype == WC_DTYPE_BF16; }

// Compute units of a device, read once.
int cus_of(int device, Check* c) {
    static std::mutex mu;
    static int held[64] = {};
    if (!c->is(device >= 0 && device < 64, "device out of range")) return 0;
    std::lock_guard<std::mutex> lk(mu);
    if (!held[device]) {
        int n = 0;
        const hipError_t e = hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, device);
        if (e != hipSuccess || n <= 0) {
            c->is(false, hipGetErrorString(e), WC_ERR_DEVICE);
            return 0;
        }
        held[device] = n;
    }
    return held[device];
}

// Runs `body` with `device` current and gives back the one that was.
template <class F>
int on_device(const char* what, int device, F&& body) {
    int before = 0;
    if (hipGetDevice(&before) != hipSuccess) return fail(WC_ERR_DEVICE, std::string(what) + ": no device");
    if (before != device && hipSetDevice(device) != hipSuccess)
        return fail(WC_ERR_DEVICE, std::string(what) + ": hipSetDevice failed");
    (void)hipGetLastError();  // an earlier caller's error is not this call's
    body();
    const hipError_t e = hipGetLastError();
    if (before != device) (void)hipSetDevice(before);
    if (e != hipSuccess) return fail(WC_ERR_DEVICE, std::string(what) + ": " + hipGetErrorString(e));
    return WC_OK;
}

template <class F>
int shielded(const char* what, F&& body) {
    try {
        return body();
    } catch (const std::exception& e) {
        return fail(WC_ERR_DEVICE, std::string(what) + ": " + e.what());
    } catch (...) {
        return fail(WC_ERR_DEVICE, std::string(what) + ": unknown exception");
    }
}

template <class A>
bool whole(const A* a, Check* c) {
    return c->is(a != nullptr, "null argument") &&
           c->is(a->bytes == sizeof(A), "the structure's size is not this library's");
}

bool finite(float x) { return x - x == 0.f; }

bool shape(int64_t rows, int64_t width, Check* c) {
    return c->is(rows >= 0 && rows < MOST, "rows out of range") &&
           c->is(width >= 1 && width < MOST_LANES, "width out of range");
}

void check(const wc_policy_args& a, Check* c) {
    if (!c->is(known(a.dtype), "unknown dtype") || !shape(a.rows, a.vocab, c)) return;
    const bool need = a.rows > 0;
    const size_t n = size_of(a.dtype);
    c->is(a.index_bits == 32 || a.index_bits == 64, "index_bits is 32 or 64");
    c->is(finite(a.inv_temperature) && a.inv_temperature > 0.f, "inv_temperature must be positive");
    c->is(a.clip_low >= 0.f && a.clip_high >= 0.f, "clip_low and clip_high must not be negative");
    c->is(finite(a.kl_coef) && finite(a.entropy_coef), "kl_coef and entropy_coef must be finite");
    c->is(!(a.ref_logp && a.ref_logits), "ref_logp and ref_logits exclude each other");
    c->matrix(a.logits, n, a.logits_stride, a.vocab, a.rows, false, need, "logits");
    c->matrix(a.legal, 1, a.legal_stride, a.vocab, a.rows, false, false, "legal");
    c->matrix(a.ref_logits, n, a.ref_stride, a.vocab, a.rows, false, false, "ref_logits");
    c->buffer(a.actions, a.index_bits / 8, need, "actions");
    c->buffer(a.behaviour_logp, 4, need, "behaviour_logp");
    c->buffer(a.advantages, 4, need, "advantages");
    c->buffer(a.weights, 4, false, "weights");
    c->buffer(a.ref_logp, 4, false, "ref_logp");
    c->buffer(a.grad_out, 4, false, "grad_out");
    c->buffer(a.loss, 4, true, "loss");
    c->buffer(a.logp, 4, need, "logp");
    c->buffer(a.kl, 4, need, "kl");
    c->buffer(a.entropy, 4, need, "entropy");
    c->matrix(a.grad, n, a.grad_stride, a.vocab, a.rows, true, false, "grad");
    c->over(a.grad, a.grad_stride, a.logits, a.logits_stride, a.rows, "grad over logits");
}

void check(const wc_preference_args& a, Check* c) {
    if (!c->is(known(a.dtype), "unknown dtype") || !shape(a.rows, a.vocab, c)) return;
    const bool need = a.rows > 0;
    const size_t n = size_of(a.dtype);
    c->is(a.pairs >= 0 && a.pairs < MOST_LANES, "pairs out of range");
    c->is(a.index_bits == 32 || a.index_bits == 64, "index_bits is 32 or 64");
    c->is(finite(a.inv_temperature) && a.inv_temperature > 0.f, "inv_temperature must be positive");
    c->is(finite(a.beta) && a.beta > 0.f, "beta must be positive");
    c->is(a.smoothing >= 0.f && a.smoothing <= 1.f, "smoothing is between 0 and 1");
    c->is(a.kind >= WC_PREFERENCE_LOGISTIC && a.kind <= WC_PREFERENCE_HINGE, "unknown kind");
    c->matrix(a.logits, n, a.logits_stride, a.vocab, a.rows, false, need, "logits");
    c->buffer(a.tokens, a.index_bits / 8, need, "tokens");
    c->buffer(a.offsets, a.index_bits / 8, a.pairs > 0, "offsets");
    c->buffer(a.ref_logp, 4, need, "ref_logp");
    c->buffer(a.weights, 4, false, "weights");
    c->buffer(a.grad_out, 4, false, "grad_out");
    c->buffer(a.loss, 4, true, "loss");
    c->buffer(a.margins, 4, a.pairs > 0, "margins");
    c->buffer(a.ratios, 4, a.pairs > 0, "ratios");
    c->buffer(a.logp, 4, need, "logp");
    c->matrix(a.grad, n, a.grad_stride, a.vocab, a.rows, true, false, "grad");
    c->over(a.grad, a.grad_stride, a.logits, a.logits_stride, a.rows, "grad over logits");
}

template <class A>
bool check_norm(const A& a, Check* c) {
    if (!c->is(known(a.dtype) && known(a.param_dtype), "unknown dtype") || !shape(a.rows, a.width, c)) return false;
    if (!c->is(a.width <= WC_NORM_MAX_WIDTH, "width beyond WC_NORM_MAX_WIDTH", WC_ERR_UNSUPPORTED)) return false;
    const size_t n = size_of(a.dtype), p = size_of(a.param_dtype);
    c->is(a.norm == WC_NORM_RMS || a.norm == WC_NORM_LAYER, "unknown norm");
    c->is(a.gate_act >= WC_GATE_NONE && a.gate_act <= WC_GATE_TANH, "unknown gate_act");
    c->is(finite(a.scale), "scale must be finite");
    c->matrix(a.block, n, a.block_stride, a.width, a.rows, false, a.rows > 0, "block");
    c->matrix(a.stream, n, a.stream_stride, a.width, a.rows, false, a.rows > 0, "stream");
    c->buffer(a.post_gain, p, false, "post_gain");
    c->buffer(a.post_bias, p, false, "post_bias");
    c->buffer(a.pre_gain, p, false, "pre_gain");
    c->matrix(a.gate, a.gate_stride ? n : p, a.gate_stride, a.width, a.rows, false, false, "gate");
    return true;
}

void check(const wc_norm_args& a, Check* c) {
    if (!check_norm(a, c)) return;
    const size_t n = size_of(a.dtype);
    c->is(a.eps >= 0.f, "eps must not be negative");
    c->buffer(a.pre_bias, size_of(a.param_dtype), false, "pre_bias");
    c->matrix(a.new_stream, n, a.new_stream_stride, a.width, a.rows, true, a.rows > 0, "new_stream");
    c->over(a.new_stream, a.new_stream_stride, a.stream, a.stream_stride, a.rows, "new_stream over stream");
    c->matrix(a.out, n, a.out_stride, a.width, a.rows, true, a.rows > 0, "out");
    c->buffer(a.stats, 16, false, "stats");
}

void check(const wc_norm_back_args& a, Check* c) {
    if (!check_norm(a, c)) return;
    const bool need = a.rows > 0;
    const size_t n = size_of(a.dtype);
    c->buffer(a.stats, 16, need, "stats");
    c->matrix(a.d_out, n, a.d_out_stride, a.width, a.rows, false, false, "d_out");
    c->matrix(a.d_new_stream, n, a.d_new_stream_stride, a.width, a.rows, false, false, "d_new_stream");
    c->matrix(a.d_block, n, a.d_block_stride, a.width, a.rows, true, need, "d_block");
    c->matrix(a.d_stream, n, a.d_stream_stride, a.width, a.rows, true, need, "d_stream");
    c->over(a.d_stream, a.d_stream_stride, a.d_new_stream, a.d_new_stream_stride, a.rows, "d_stream over d_new_stream");
    c->buffer(a.d_post_gain, 4, false, "d_post_gain");
    c->buffer(a.d_post_bias, 4, false, "d_post_bias");
    c->buffer(a.d_pre_gain, 4, false, "d_pre_gain");
    c->buffer(a.d_pre_bias, 4, false, "d_pre_bias");
    if (a.d_gate) {
        c->is(a.gate != nullptr, "d_gate without a gate");
        if (a.gate_stride) c->matrix(a.d_gate, n, a.d_gate_stride, a.width, a.rows, true, true, "d_gate");
        else c->buffer(a.d_gate, 4, true, "d_gate");
    }
}

enum class Ckpt { write, read, back };

void check(const wc_ckpt_args& a, Ckpt use, Check* c) {
    if (!c->is(known(a.dtype), "unknown dtype") || !shape(a.rows, a.width, c)) return;
    const bool need = a.rows > 0;
    const size_t n = size_of(a.dtype);
    c->is(a.act >= WC_ACT_NONE && a.act <= WC_ACT_SILU, "unknown act");
    const bool write = use == Ckpt::write;
    c->matrix(a.q, 1, a.q_stride, a.width, a.rows, write, need, "q");
    c->matrix(a.exps, 1, a.exps_stride, (a.width + WC_CKPT_GROUP - 1) / WC_CKPT_GROUP, a.rows, write, need, "exps");
    if (use != Ckpt::read) c->matrix(a.x, n, a.x_stride, a.width, a.rows, false, need, "x");
    c->matrix(a.y, n, a.y_stride, a.width, a.rows, true, need && !write, "y");
    if (use == Ckpt::back) c->over(a.y, a.y_stride, a.x, a.x_stride, a.rows, "y over x");
}

void check(const wc_ckpt_weight_args& a, Check* c) {
    if (!c->is(known(a.dtype), "unknown dtype") || !shape(a.rows, a.width, c) || !shape(a.rows, a.out, c)) return;
    const bool need = a.rows > 0;
    c->is(a.width < (1 << 20) && a.out < (1 << 20), "width or out beyond 2^20", WC_ERR_UNSUPPORTED);
    c->is(a.act >= WC_ACT_NONE && a.act <= WC_ACT_SILU, "unknown act");
    c->is(a.dtype != WC_DTYPE_F32 || a.act == WC_ACT_NONE || a.act == WC_ACT_RELU,
          "a float32 gradient takes no activation but relu", WC_ERR_UNSUPPORTED);
    c->is(a.weight_dtype == WC_DTYPE_F32 || a.weight_dtype == a.dtype, "weight_dtype is float32 or the gradient's");
    c->matrix(a.q, 1, a.q_stride, a.width, a.rows, false, need, "q");
    c->matrix(a.exps, 1, a.exps_stride, (a.width + WC_CKPT_GROUP - 1) / WC_CKPT_GROUP, a.rows, false, need, "exps");
    c->matrix(a.grad, size_of(a.dtype), a.grad_stride, a.out, a.rows, false, need, "grad");
    c->matrix(a.weight, size_of(a.weight_dtype), a.weight_stride, a.out, a.width, true, true, "weight");
    c->buffer(a.bias, 4, false, "bias");
}

// What both directions of a layer have.
template <class A>
bool check_layer(const A& a, Check* c) {
    if (!c->is(known(a.dtype), "unknown dtype") || !shape(a.rows, a.width, c) || !shape(a.rows, a.out, c)) return false;
    if (!c->is(a.rows < MOST_LANES, "rows beyond 2^31", WC_ERR_UNSUPPORTED) ||
        !c->is(a.width <= (1 << 20) && a.out <= (1 << 20), "width or out beyond 2^20", WC_ERR_UNSUPPORTED))
        return false;
    c->is(a.weight_layout == WC_WEIGHT_IN_OUT || a.weight_layout == WC_WEIGHT_OUT_IN, "unknown weight_layout");
    c->is(a.act >= WC_ACT_NONE && a.act <= WC_ACT_SILU, "unknown act");
    return true;
}

template <class A>
void check_weight(const A& a, const void* p, size_t n, int64_t stride, bool written, bool need, const char* name, Check* c) {
    const bool io = a.weight_layout == WC_WEIGHT_IN_OUT;
    c->matrix(p, n, stride, io ? a.out : a.width, io ? a.width : a.out, written, need, name);
}

void check(const wc_linear_args& a, Check* c) {
    if (!check_layer(a, c)) return;
    const size_t n = size_of(a.dtype);
    const bool need = a.rows > 0;
    c->is(a.bias_dtype == WC_DTYPE_F32 || a.bias_dtype == a.dtype, "bias_dtype is float32 or the matrices'");
    c->matrix(a.x, n, a.x_stride, a.width, a.rows, false, need, "x");
    check_weight(a, a.weight, n, a.weight_stride, false, need, "weight", c);
    c->buffer(a.bias, known(a.bias_dtype) ? size_of(a.bias_dtype) : 4, false, "bias");
    c->matrix(a.residual, n, a.residual_stride, a.out, a.rows, false, false, "residual");
    c->matrix(a.pre, 4, a.pre_stride, a.out, a.rows, true, false, "pre");
    c->matrix(a.y, n, a.y_stride, a.out, a.rows, true, need, "y");
    c->over(a.y, a.y_stride, a.residual, a.residual_stride, a.rows, "y over residual");
}

void check(const wc_linear_back_args& a, Check* c) {
    if (!check_layer(a, c)) return;
    const size_t n = size_of(a.dtype);
    const bool need = a.rows > 0;
    c->is(a.grad_dtype == WC_DTYPE_F32 || a.grad_dtype == a.dtype, "grad_dtype is float32 or the matrices'");
    c->matrix(a.d_out, n, a.d_out_stride, a.out, a.rows, false, need, "d_out");
    if (a.act != WC_ACT_NONE) c->matrix(a.pre, 4, a.pre_stride, a.out, a.rows, false, need, "pre");
    if (a.d_weight) {
        c->matrix(a.x, n, a.x_stride, a.width, a.rows, false, need, "x");
        check_weight(a, a.d_weight, known(a.grad_dtype) ? size_of(a.grad_dtype) : 4, a.d_weight_stride, true, true,
                     "d_weight", c);
    }
    if (a.d_x) {
        check_weight(a, a.weight, n, a.weight_stride, false, need, "weight", c);
        c->matrix(a.d_x, n, a.d_x_stride, a.width, a.rows, true, need, "d_x");
    }
    c->buffer(a.d_bias, 4, false, "d_bias");
}

void check(const wc_orthogonalise_args& a, Check* c) {
    if (!c->is(known(a.dtype) && known(a.out_dtype), "unknown dtype")) return;
    c->is(a.batch >= 0 && a.batch <= 65535, "batch is 0 to 65535");
    c->is(a.rows >= 1 && a.width >= 1, "rows and width are at least 1");
    if (!c->is(a.rows <= (1 << 20) && a.width <= (1 << 20), "rows or width beyond 2^20", WC_ERR_UNSUPPORTED)) return;
    c->is(a.steps >= 1 && a.steps <= 64, "steps is 1 to 64");
    c->is(finite(a.a) && finite(a.b) && finite(a.c) && finite(a.scale), "coefficients and scale must be finite");
    c->is(finite(a.eps) && a.eps >= 0.f, "eps must not be negative");
    const size_t n = size_of(a.dtype), o = size_of(a.out_dtype);
    c->matrix(a.update, n, a.update_stride, a.width, a.rows, false, a.batch > 0, "update");
    c->matrix(a.out, o, a.out_stride, a.width, a.rows, true, a.batch > 0, "out");
    // a matrix's own rows are apart already; matrices follow each other, or lie between each other's rows
    const int64_t deep = (a.rows - 1) * a.out_stride + a.width;
    c->is(a.batch <= 1 || (a.update_batch >= 0 && a.update_batch <= MOST), "update_batch out of range");
    c->is(a.batch <= 1 || (a.out_batch >= deep && a.out_batch <= MOST), "out's matrices overlap");
    // one matrix is read whole before its result is written; of several, each only before its own
    if (a.out && a.out == a.update && a.batch > 1)
        c->is(a.out_dtype == a.dtype && a.out_batch == a.update_batch && (a.rows <= 1 || a.out_stride == a.update_stride),
              "out over update itself needs its type and its strides");
}

template <class A>
bool check_logits(const A& a, Check* c) {
    if (!c->is(known(a.dtype), "unknown dtype") || !shape(a.rows, a.vocab, c)) return false;
    if (!c->is(a.rows < MOST_LANES && a.rows * ((a.vocab + 1023) / 1024) < MOST_LANES, "more rows of this length than a launch holds",
               WC_ERR_UNSUPPORTED))
        return false;
    c->is(a.index_bits == 32 || a.index_bits == 64, "index_bits is 32 or 64");
    c->is(finite(a.inv_temperature) && a.inv_temperature > 0.f, "inv_temperature must be positive");
    c->matrix(a.logits, size_of(a.dtype), a.logits_stride, a.vocab, a.rows, false, a.rows > 0, "logits");
    c->matrix(a.legal, 1, a.legal_stride, a.vocab, a.rows, false, false, "legal");
    c->buffer(a.tokens, a.index_bits == 32 ? 4 : 8, false, "tokens");
    return true;
}

void check(const wc_logp_args& a, Check* c) {
    if (!check_logits(a, c)) return;
    const bool need = a.rows > 0;
    c->is(a.top >= 0 && a.top <= WC_TOP_MAX, "top is 0 to 64");
    c->buffer(a.logp, 4, need && a.tokens, "logp");
    c->buffer(a.rank, 4, need && a.tokens, "rank");
    c->buffer(a.entropy, 4, need, "entropy");
    c->buffer(a.top_logp, 4, need && a.top, "top_logp");
    c->buffer(a.top_index, 4, need && a.top, "top_index");
    c->buffer(a.stats, 16, false, "stats");
}

void check(const wc_logp_back_args& a, Check* c) {
    if (!check_logits(a, c)) return;
    c->buffer(a.stats, 16, a.rows > 0, "stats");
    c->buffer(a.d_logp, 4, false, "d_logp");
    c->buffer(a.d_entropy, 4, false, "d_entropy");
    c->matrix(a.grad, size_of(a.dtype), a.grad_stride, a.vocab, a.rows, true, a.rows > 0, "grad");
    c->over(a.grad, a.grad_stride, a.logits, a.logits_stride, a.rows, "grad over logits");
}

template <class A>
void workspace(const A& a, size_t want, Check* c) {
    c->is(a.workspace_bytes >= want && (a.workspace || !want), "the workspace is too small");
    c->is(c->aligned(a.workspace, 256), "the workspace is not 256-byte aligned");
}

// One entry point that needs scratch: `run` false writes its size only.
template <class A, class S, class L>
int with_scratch(const char* what, const A* a, uint64_t* bytes, S&& scratch, L&& launch, void* stream) {
    return shielded(what, [&]() -> int {
        Check c{what};
        if (whole(a, &c)) check(*a, &c);
        const int cus = c.code == WC_OK ? cus_of(a->device, &c) : 0;
        if (c.code != WC_OK) return fail(c.code, c.msg);
        const size_t want = scratch(*a, cus);
        if (bytes) {
            *bytes = want;
            return WC_OK;
        }
        workspace(*a, want, &c);
        if (c.code != WC_OK) return fail(c.code, c.msg);
        return on_device(what, a->device, [&] { launch(*a, cus, (hipStream_t)stream); });
    });
}

template <class L>
int ckpt(const char* what, const wc_ckpt_args* a, Ckpt use, L&& launch, void* stream) {
    return shielded(what, [&]() -> int {
        Check c{what};
        if (whole(a, &c)) check(*a, use, &c);
        const int cus = c.code == WC_OK ? cus_of(a->device, &c) : 0;
        if (c.code != WC_OK) return fail(c.code, c.msg);
        return on_device(what, a->device, [&] { launch(*a, cus, (hipStream_t)stream); });
    });
}

}  // namespace

extern "C" {

int wc_policy_workspace(const wc_policy_args* a, uint64_t* bytes) {
    if (!bytes) return fail(WC_ERR_INVALID, "wc_policy_workspace: null argument");
    return with_scratch("wc_policy_workspace", a, bytes, learn::policy_scratch, learn::launch_policy, nullptr);
}
int wc_policy_loss(const wc_policy_args* a, void* stream) {
    return with_scratch("wc_policy_loss", a, nullptr, learn::policy_scratch, learn::launch_policy, stream);
}

int wc_preference_workspace(const wc_preference_args* a, uint64_t* bytes) {
    if (!bytes) return fail(WC_ERR_INVALID, "wc_preference_workspace: null argument");
    return with_scratch("wc_preference_workspace", a, bytes, learn::preference_scratch, learn::launch_preference,
                        nullptr);
}
int wc_preference_loss(const wc_preference_args* a, void* stream) {
    return with_scratch("wc_preference_loss", a, nullptr, learn::preference_scratch, learn::launch_preference, stream);
}

int wc_residual_norm(const wc_norm_args* a, void* stream) {
    return shielded("wc_residual_norm", [&]() -> int {
        Check c{"wc_residual_norm"};
        if (whole(a, &c)) check(*a, &c);
        const int cus = c.code == WC_OK ? cus_of(a->device, &c) : 0;
        if (c.code != WC_OK) return fail(c.code, c.msg);
        return on_device("wc_residual_norm", a->device, [&] { learn::launch_norm(*a, cus, (hipStream_t)stream); });
    });
}

int wc_residual_norm_workspace(const wc_norm_back_args* a, uint64_t* bytes) {
    if (!bytes) return fail(WC_ERR_INVALID, "wc_residual_norm_workspace: null argument");
    return with_scratch("wc_residual_norm_workspace", a, bytes, learn::norm_back_scratch, learn::launch_norm_back,
                        nullptr);
}
int wc_residual_norm_backward(const wc_norm_back_args* a, void* stream) {
    return with_scratch("wc_residual_norm_backward", a, nullptr, learn::norm_back_scratch, learn::launch_norm_back,
                        stream);
}

int wc_ckpt_write(const wc_ckpt_args* a, void* stream) {
    return ckpt("wc_ckpt_write", a, Ckpt::write, learn::launch_ckpt_write, stream);
}
int wc_ckpt_read(const wc_ckpt_args* a, void* stream) {
    return ckpt("wc_ckpt_read", a, Ckpt::read, learn::launch_ckpt_read, stream);
}
int wc_ckpt_act_backward(const wc_ckpt_args* a, void* stream) {
    return ckpt("wc_ckpt_act_backward", a, Ckpt::back, learn::launch_ckpt_act_back, stream);
}

int wc_ckpt_weight_workspace(const wc_ckpt_weight_args* a, uint64_t* bytes) {
    if (!bytes) return fail(WC_ERR_INVALID, "wc_ckpt_weight_workspace: null argument");
    return with_scratch("wc_ckpt_weight_workspace", a, bytes, learn::ckpt_weight_scratch, learn::launch_ckpt_weight,
                        nullptr);
}
int wc_ckpt_weight_grad(const wc_ckpt_weight_args* a, void* stream) {
    return with_scratch("wc_ckpt_weight_grad", a, nullptr, learn::ckpt_weight_scratch, learn::launch_ckpt_weight,
                        stream);
}

int wc_linear_workspace(const wc_linear_args* a, uint64_t* bytes) {
    if (!bytes) return fail(WC_ERR_INVALID, "wc_linear_workspace: null argument");
    return with_scratch("wc_linear_workspace", a, bytes, learn::linear_scratch, learn::launch_linear, nullptr);
}
int wc_linear(const wc_linear_args* a, void* stream) {
    return with_scratch("wc_linear", a, nullptr, learn::linear_scratch, learn::launch_linear, stream);
}

int wc_linear_backward_workspace(const wc_linear_back_args* a, uint64_t* bytes) {
    if (!bytes) return fail(WC_ERR_INVALID, "wc_linear_backward_workspace: null argument");
    return with_scratch("wc_linear_backward_workspace", a, bytes, learn::linear_back_scratch, learn::launch_linear_back, nullptr);
}
int wc_linear_backward(const wc_linear_back_args* a, void* stream) {
    return with_scratch("wc_linear_backward", a, nullptr, learn::linear_back_scratch, learn::launch_linear_back, stream);
}

int wc_orthogonalise_workspace(const wc_orthogonalise_args* a, uint64_t* bytes) {
    if (!bytes) return fail(WC_ERR_INVALID, "wc_orthogonalise_workspace: null argument");
    return with_scratch("wc_orthogonalise_workspace", a, bytes, learn::orthogonalise_scratch, learn::launch_orthogonalise, nullptr);
}
int wc_orthogonalise(const wc_orthogonalise_args* a, void* stream) {
    return with_scratch("wc_orthogonalise", a, nullptr, learn::orthogonalise_scratch, learn::launch_orthogonalise, stream);
}

int wc_token_logp_workspace(const wc_logp_args* a, uint64_t* bytes) {
    if (!bytes) return fail(WC_ERR_INVALID, "wc_token_logp_workspace: null argument");
    return with_scratch("wc_token_logp_workspace", a, bytes, learn::logp_scratch, learn::launch_logp, nullptr);
}
int wc_token_logp(const wc_logp_args* a, void* stream) {
    return with_scratch("wc_token_logp", a, nullptr, learn::logp_scratch, learn::launch_logp, stream);
}

int wc_token_logp_backward(const wc_logp_back_args* a, void* stream) {
    return shielded("wc_token_logp_backward", [&]() -> int {
        Check c{"wc_token_logp_backward"};
        if (whole(a, &c)) check(*a, &c);
        const int cus = c.code == WC_OK ? cus_of(a->device, &c) : 0;
        if (c.code != WC_OK) return fail(c.code, c.msg);
        return on_device("wc_token_logp_backward", a->device,
                         [&] { learn::launch_logp_back(*a, cus, (hipStream_t)stream); });
    });
}

}  // extern "C"
