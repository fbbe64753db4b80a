// capi_block.cpp -- the extern "C" entry points for transformer layers
// (include/acfun/acfun.h): MXFP4 quantizer and products, norms around a block.
// Arguments are checked before the device is touched; nothing is written when
// a call is refused, and no C++ exception leaves an entry.
#include <exception>

#include "../../include/acfun/acfun.h"
#include "mx.hpp"

using namespace acfun;

namespace {

// The first failed check of a call is its error.
struct Checks {
    const char* who;
    bool ok = true;
    Checks& need(bool good, const char* what) {
        if (ok && !good) {
            set_error("%s: %s", who, what);
            ok = false;
        }
        return *this;
    }
    Checks& type(int t) { return need(type_ok(t), "type is not ACFUN_F32, ACFUN_BF16 or ACFUN_F16"); }
    Checks& act(int a) { return need(a == 0 || a == 1, "act is not 0 or 1"); }
    // a float tensor: aligned to its elements
    Checks& tensor(const void* p, int t, const char* what) {
        need(p != nullptr, what);
        return need(!type_ok(t) || (uintptr_t)p % type_size(t) == 0, "a tensor is not aligned to its elements");
    }
    // what is written is apart from what is read: workgroups read it at any time
    Checks& apart(const void* out, size_t n, const void* in, size_t m) {
        const uintptr_t o = (uintptr_t)out, i = (uintptr_t)in;
        return need(!in || o + n <= i || i + m <= o, "a result overlaps an input");
    }
    // or it is the same buffer, of which every element is read before it is written
    Checks& apart_or_same(const void* out, const void* in, size_t n) {
        return out == in ? *this : apart(out, n, in, n);
    }
    Checks& param(const float* p) { return need((uintptr_t)p % 4 == 0, "a parameter is not aligned to 4 bytes"); }
    Checks& fits(bool f) { return need(f, "too large: a launch holds fewer than 2^32 threads"); }
    Checks& held(const uint8_t* codes, const uint8_t* scales) {
        need(codes && scales, "codes or scales are NULL");
        return need((uintptr_t)codes % 16 == 0 && (uintptr_t)scales % 16 == 0,
                    "codes or scales are not aligned to 16 bytes");
    }
};

// Runs f, which returns false with the error set; an exception becomes one.
template <class F>
int call(const char* who, F f) {
    try {
        return ensure_device() && f() ? 0 : -1;
    } catch (const std::exception& e) {
        set_error("%s: %s", who, e.what());
    } catch (...) {
        set_error("%s: exception", who);
    }
    return -1;
}

// A host-pointer call: staged operands, synchronized at the end.
template <class F>
void staged(const char* who, F f) {
    (void)call(who, [&] {
        HostCall hc(lib_stream());
        const bool ok = f(hc) && !hc.failed();
        if (!ok) {
            (void)hipStreamSynchronize(hc.stream());
            return false;
        }
        return hc.finish();
    });
}

}  // namespace

extern "C" {

// ------------------------------------------------------------------ MXFP4
size_t acfun_mxfp4_code_bytes(int rows, int K) { return rows > 0 && K > 0 ? mx_code_bytes(rows, K) : 0; }
size_t acfun_mxfp4_scale_bytes(int rows, int K) { return rows > 0 && K > 0 ? mx_scale_bytes(rows, K) : 0; }

int acfun_dev_quantize_mxfp4(const void* x, int type, int rows, int K, int trans, uint8_t* codes,
                             uint8_t* scales, void* stream) {
    Checks c{"acfun_dev_quantize_mxfp4"};
    if (!c.type(type).need(rows >= 0 && K >= 0, "a size is negative").ok) return -1;
    if (rows == 0 || K == 0) return 0;
    if (!c.tensor(x, type, "x is NULL").held(codes, scales).ok) return -1;
    const size_t n = (size_t)rows * K * type_size(type);
    c.apart(codes, mx_code_bytes(rows, K), x, n).apart(scales, mx_scale_bytes(rows, K), x, n);
    c.apart(codes, mx_code_bytes(rows, K), scales, mx_scale_bytes(rows, K));
    if (!c.fits(mx_quant_fits(rows, K, trans)).ok) return -1;
    return call(c.who, [&] { return mx_quantize(x, type, rows, K, trans, codes, scales, resolve(stream)); });
}

int acfun_dev_dequantize_mxfp4(const uint8_t* codes, const uint8_t* scales, int rows, int K, void* x, int type,
                               void* stream) {
    Checks c{"acfun_dev_dequantize_mxfp4"};
    if (!c.type(type).need(rows >= 0 && K >= 0, "a size is negative").ok) return -1;
    if (rows == 0 || K == 0) return 0;
    if (!c.tensor(x, type, "x is NULL").held(codes, scales).ok) return -1;
    const size_t n = (size_t)rows * K * type_size(type);
    if (!c.apart(x, n, codes, mx_code_bytes(rows, K)).apart(x, n, scales, mx_scale_bytes(rows, K)).ok) return -1;
    if (!c.fits(mx_quant_fits(rows, K, 0)).ok) return -1;
    return call(c.who, [&] { return mx_dequantize(codes, scales, rows, K, x, type, resolve(stream)); });
}

int acfun_dev_gemm_mxfp4(int M, int N, int K, const uint8_t* A, const uint8_t* a_scales, const uint8_t* B,
                         const uint8_t* b_scales, void* C, int type, const float* bias, int act, void* stream) {
    Checks c{"acfun_dev_gemm_mxfp4"};
    if (!c.type(type).act(act).need(M >= 0 && N >= 0 && K >= 0, "a size is negative").ok) return -1;
    if (M == 0 || N == 0) return 0;
    if (K > 0) c.held(A, a_scales).held(B, b_scales);
    if (!c.tensor(C, type, "C is NULL").param(bias).ok) return -1;
    const size_t n = (size_t)M * N * type_size(type);
    if (K > 0) {
        c.apart(C, n, A, mx_code_bytes(M, K)).apart(C, n, a_scales, mx_scale_bytes(M, K));
        c.apart(C, n, B, mx_code_bytes(N, K)).apart(C, n, b_scales, mx_scale_bytes(N, K));
    }
    if (!c.apart(C, n, bias, 4 * (size_t)N).fits(mm_fits(M, N, K)).ok) return -1;
    return call(c.who, [&] {
        return mx_gemm(M, N, K, A, a_scales, B, b_scales, C, type, bias, act, resolve(stream));
    });
}

int acfun_dev_fc_mxfp4(const void* input, int type, int N, int Cin, const uint8_t* weight, const uint8_t* wscale,
                       const float* bias, int Cout, void* output, int act, void* stream) {
    Checks c{"acfun_dev_fc_mxfp4"};
    if (!c.type(type).act(act).need(N >= 0 && Cin >= 0 && Cout >= 0, "a size is negative").ok) return -1;
    if (N == 0 || Cout == 0) return 0;
    if (Cin > 0) c.tensor(input, type, "input is NULL").held(weight, wscale);
    if (!c.tensor(output, type, "output is NULL").param(bias).ok) return -1;
    const size_t n = (size_t)N * Cout * type_size(type);
    if (Cin > 0) {
        c.apart(output, n, input, (size_t)N * Cin * type_size(type));
        c.apart(output, n, weight, mx_code_bytes(Cout, Cin)).apart(output, n, wscale, mx_scale_bytes(Cout, Cin));
    }
    if (!c.apart(output, n, bias, 4 * (size_t)Cout).fits(fc_fits(N, Cout, Cin)).ok) return -1;
    return call(c.who, [&] {
        return mx_fc(input, type, N, Cin, weight, wscale, bias, Cout, output, act, resolve(stream));
    });
}

void acfun_quantize_weights_mxfp4(const float* w, int K, int N, uint8_t* codes, uint8_t* scales) {
    if (K <= 0 || N <= 0) return;
    Checks c{"acfun_quantize_weights_mxfp4"};
    if (!c.need(w && codes && scales, "a pointer is NULL").ok) return;
    staged(c.who, [&](HostCall& hc) {
        auto dw = (const float*)hc.in(w, (size_t)K * N * sizeof(float));
        auto dc = (uint8_t*)hc.out(codes, mx_code_bytes(N, K));
        auto ds = (uint8_t*)hc.out(scales, mx_scale_bytes(N, K));
        return !hc.failed() && acfun_dev_quantize_mxfp4(dw, ACFUN_F32, N, K, 1, dc, ds, hc.stream()) == 0;
    });
}

void acfun_fc_mxfp4(const float* input, int N, int Cin, const uint8_t* weight, const uint8_t* wscale,
                    const float* bias, int Cout, float* output, int act) {
    if (N <= 0 || Cin < 0 || Cout <= 0) return;
    Checks c{"acfun_fc_mxfp4"};
    if (!c.need(output && (Cin == 0 || (input && weight && wscale)), "a pointer is NULL").ok) return;
    staged(c.who, [&](HostCall& hc) {
        auto dx = (const float*)hc.in(input, (size_t)N * Cin * sizeof(float));
        auto dw = (const uint8_t*)hc.in(weight, acfun_mxfp4_code_bytes(Cout, Cin));
        auto ds = (const uint8_t*)hc.in(wscale, acfun_mxfp4_scale_bytes(Cout, Cin));
        auto db = (const float*)hc.in(bias, (size_t)Cout * sizeof(float));
        auto dy = (float*)hc.out(output, (size_t)N * Cout * sizeof(float));
        return !hc.failed() &&
               acfun_dev_fc_mxfp4(dx, ACFUN_F32, N, Cin, dw, ds, db, Cout, dy, act, hc.stream()) == 0;
    });
}

// ------------------------------------------------------------------ norms
int acfun_dev_norm(const void* x, int type, int rows, int cols, int kind, const float* weight,
                   const float* bias, float eps, void* h, void* stream) {
    Checks c{"acfun_dev_norm"};
    if (!c.type(type).need(rows >= 0 && cols >= 0, "a size is negative").ok) return -1;
    if (rows == 0 || cols == 0) return 0;
    c.need(cols <= kNormMaxCols, "more than 32768 columns");
    c.need(kind == ACFUN_RMSNORM || kind == ACFUN_LAYERNORM, "kind is not ACFUN_RMSNORM or ACFUN_LAYERNORM");
    c.need(eps >= 0.f, "eps is negative");
    c.tensor(x, type, "x is NULL").tensor(h, type, "h is NULL").param(weight).param(bias);
    if (!c.ok) return -1;
    const size_t n = (size_t)rows * cols * type_size(type), np = 4 * (size_t)cols;
    if (!c.apart_or_same(h, x, n).apart(h, n, weight, np).apart(h, n, bias, np).ok) return -1;
    NormArgs a{nullptr, x, rows, cols, kind, nullptr, nullptr, nullptr, 1, 1.f, weight, bias, eps, nullptr, h};
    return call(c.who, [&] { return norm_rows(a, type, resolve(stream)); });
}

int acfun_dev_norm_residual(const void* y, const void* x, int type, int rows, int cols, int kind,
                            const float* post_w, const float* post_b, const void* gate, int gate_group,
                            float res_scale, const float* pre_w, const float* pre_b, float eps, void* x_out,
                            void* h, void* stream) {
    Checks c{"acfun_dev_norm_residual"};
    if (!c.type(type).need(rows >= 0 && cols >= 0, "a size is negative").ok) return -1;
    if (rows == 0 || cols == 0) return 0;
    c.need(cols <= kNormMaxCols, "more than 32768 columns");
    c.need(kind == ACFUN_RMSNORM || kind == ACFUN_LAYERNORM, "kind is not ACFUN_RMSNORM or ACFUN_LAYERNORM");
    c.need(eps >= 0.f, "eps is negative");
    c.need(!gate || gate_group > 0, "gate_group is not positive");
    c.tensor(y, type, "y is NULL").tensor(x, type, "x is NULL").tensor(x_out, type, "x_out is NULL");
    if (gate) c.tensor(gate, type, "");
    if (h) c.tensor(h, type, "");
    c.param(post_w).param(post_b).param(pre_w).param(pre_b);
    c.need(h != x_out, "h and x_out are the same buffer");
    if (!c.ok) return -1;
    const size_t n = (size_t)rows * cols * type_size(type), np = 4 * (size_t)cols;
    const size_t ng = gate ? ((size_t)rows + gate_group - 1) / gate_group * cols * type_size(type) : 0;
    c.apart(x_out, n, h, h ? n : 0);
    for (void* out : {x_out, h}) {
        if (!out) continue;
        c.apart_or_same(out, x, n).apart_or_same(out, y, n).apart(out, n, gate, ng);
        for (const float* q : {post_w, post_b, pre_w, pre_b}) c.apart(out, n, q, np);
    }
    if (!c.ok) return -1;
    NormArgs a{y, x, rows, cols, kind, post_w, post_b, gate, gate ? gate_group : 1, res_scale, pre_w, pre_b, eps,
               x_out, h};
    return call(c.who, [&] { return norm_rows(a, type, resolve(stream)); });
}

}  // extern "C"
