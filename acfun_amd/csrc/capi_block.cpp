// capi_block.cpp -- the extern "C" entry points for transformer layers
// (include/acfun/acfun.h): MXFP4 and Q8 quantizers and products, norms around a block,
// sampling.
// Arguments are checked before the device is touched; nothing is written when
// a call is refused, and no C++ exception leaves an entry.
#include <exception>

#include "../../include/acfun/acfun.h"
#include "q8.hpp"

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
    Checks& param(const int* p) { return param((const float*)p); }
    Checks& fits(bool f) { return need(f, "too large: a launch holds fewer than 2^32 threads"); }
    Checks& held(const void* codes, const void* scales) {
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

constexpr const char* kQ8Long = "K is more than 131072: sums of products could pass 32 bits";

// A product of Q8 operands, or (rows) a layer on float rows.
int q8_product(const char* who, const Q8Product& p, int type, bool rows, void* stream) {
    Checks c{who};
    c.type(type).need(p.act >= 0 && p.act <= ACFUN_GELU_TANH, "act is not 0 or one of ACFUN_RELU to ACFUN_GELU_TANH");
    if (!c.need(p.M >= 0 && p.N >= 0 && p.K >= 0, "a size is negative").ok) return -1;
    if (p.M == 0 || p.N == 0) return 0;
    c.need(p.K <= kQ8MaxK, kQ8Long);
    const int mats = p.gated ? 2 : 1;
    const size_t n = (size_t)p.M * p.N * type_size(type);
    if (p.K > 0) {
        if (rows) c.tensor(p.A, type, "input is NULL");
        else c.held(p.A, p.As);
        for (int g = 0; g < mats; ++g) c.held(p.B[g], p.Bs[g]);
    }
    c.tensor(p.C, type, "the result is NULL");
    for (int g = 0; g < mats; ++g) c.param(p.bias[g]);
    if (!c.ok) return -1;
    if (p.K > 0) {
        if (rows) c.apart(p.C, n, p.A, (size_t)p.M * p.K * type_size(type));
        else c.apart(p.C, n, p.A, q8_code_bytes(p.M, p.K)).apart(p.C, n, p.As, q8_scale_bytes(p.M));
        for (int g = 0; g < mats; ++g)
            c.apart(p.C, n, p.B[g], q8_code_bytes(p.N, p.K)).apart(p.C, n, p.Bs[g], q8_scale_bytes(p.N));
    }
    for (int g = 0; g < mats; ++g) c.apart(p.C, n, p.bias[g], 4 * (size_t)p.N);
    if (!c.fits(q8_mm_fits(p.M, p.N, p.K, p.gated) && (!rows || q8_quant_fits(p.M, 0))).ok) return -1;
    return call(who, [&] { return rows ? q8_fc(who, p, type, resolve(stream)) : q8_gemm(p, type, resolve(stream)); });
}

// A layer on host or device pointers, fp32.
void q8_host_layer(Checks c, Q8Product p) {
    if (p.M <= 0 || p.K < 0 || p.N <= 0) return;
    const int mats = p.gated ? 2 : 1;
    c.need(p.C && (p.K == 0 || p.A), "a pointer is NULL");
    for (int g = 0; g < mats; ++g) c.need(p.K == 0 || (p.B[g] && p.Bs[g]), "a pointer is NULL");
    if (!c.ok) return;
    staged(c.who, [&](HostCall& hc) {
        p.A = hc.in(p.A, (size_t)p.M * p.K * sizeof(float));
        for (int g = 0; g < mats; ++g) {
            p.B[g] = (const int8_t*)hc.in(p.B[g], acfun_q8_code_bytes(p.N, p.K));
            p.Bs[g] = (const float*)hc.in(p.Bs[g], q8_scale_bytes(p.N));
            p.bias[g] = (const float*)hc.in(p.bias[g], (size_t)p.N * sizeof(float));
        }
        p.C = hc.out(p.C, (size_t)p.M * p.N * sizeof(float));
        return !hc.failed() && q8_product(c.who, p, ACFUN_F32, true, hc.stream()) == 0;
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

// ------------------------------------------------------------------ Q8
size_t acfun_q8_code_bytes(int rows, int K) { return rows > 0 && K > 0 ? q8_code_bytes(rows, K) : 0; }
size_t acfun_q8_scale_bytes(int rows) { return rows > 0 ? q8_scale_bytes(rows) : 0; }

int acfun_dev_quantize_q8(const void* x, int type, int rows, int K, int trans, int8_t* codes, float* scales,
                          void* stream) {
    Checks c{"acfun_dev_quantize_q8"};
    if (!c.type(type).need(rows >= 0 && K >= 0, "a size is negative").ok) return -1;
    if (rows == 0 || K == 0) return 0;
    c.need(K <= kQ8MaxK, kQ8Long);
    if (!c.tensor(x, type, "x is NULL").held(codes, scales).ok) return -1;
    const size_t n = (size_t)rows * K * type_size(type);
    c.apart(codes, q8_code_bytes(rows, K), x, n).apart(scales, q8_scale_bytes(rows), x, n);
    c.apart(codes, q8_code_bytes(rows, K), scales, q8_scale_bytes(rows));
    if (!c.fits(q8_quant_fits(rows, trans)).ok) return -1;
    return call(c.who, [&] { return q8_quantize(x, type, rows, K, trans, codes, scales, resolve(stream)); });
}

int acfun_dev_dequantize_q8(const int8_t* codes, const float* scales, int rows, int K, void* x, int type,
                            void* stream) {
    Checks c{"acfun_dev_dequantize_q8"};
    if (!c.type(type).need(rows >= 0 && K >= 0, "a size is negative").ok) return -1;
    if (rows == 0 || K == 0) return 0;
    c.need(K <= kQ8MaxK, kQ8Long);
    if (!c.tensor(x, type, "x is NULL").held(codes, scales).ok) return -1;
    const size_t n = (size_t)rows * K * type_size(type);
    if (!c.apart(x, n, codes, q8_code_bytes(rows, K)).apart(x, n, scales, q8_scale_bytes(rows)).ok) return -1;
    if (!c.fits(q8_dequant_fits(rows, K)).ok) return -1;
    return call(c.who, [&] { return q8_dequantize(codes, scales, rows, K, x, type, resolve(stream)); });
}

int acfun_dev_gemm_q8(int M, int N, int K, const int8_t* A, const float* a_scales, const int8_t* B,
                      const float* b_scales, void* C, int type, const float* bias, int act, void* stream) {
    return q8_product("acfun_dev_gemm_q8", {M, N, K, A, a_scales, {B}, {b_scales}, {bias}, C, act, false}, type, false,
                      stream);
}

int acfun_dev_fc_q8(const void* input, int type, int N, int Cin, const int8_t* weight, const float* wscale,
                    const float* bias, int Cout, void* output, int act, void* stream) {
    return q8_product("acfun_dev_fc_q8", {N, Cout, Cin, input, nullptr, {weight}, {wscale}, {bias}, output, act, false},
                      type, true, stream);
}

int acfun_dev_gemm_gated_q8(int M, int N, int K, const int8_t* A, const float* a_scales, const int8_t* G,
                            const float* g_scales, const int8_t* U, const float* u_scales, void* C, int type,
                            const float* gbias, const float* ubias, int act, void* stream) {
    return q8_product("acfun_dev_gemm_gated_q8",
                      {M, N, K, A, a_scales, {G, U}, {g_scales, u_scales}, {gbias, ubias}, C, act, true}, type, false,
                      stream);
}

int acfun_dev_fc_gated_q8(const void* input, int type, int N, int Cin, const int8_t* gate, const float* gscale,
                          const float* gbias, const int8_t* up, const float* uscale, const float* ubias, int Cout,
                          void* output, int act, void* stream) {
    return q8_product("acfun_dev_fc_gated_q8",
                      {N, Cout, Cin, input, nullptr, {gate, up}, {gscale, uscale}, {gbias, ubias}, output, act, true},
                      type, true, stream);
}

void acfun_quantize_weights_q8(const float* w, int K, int N, int8_t* codes, float* scales) {
    if (K <= 0 || N <= 0) return;
    Checks c{"acfun_quantize_weights_q8"};
    if (!c.need(w && codes && scales, "a pointer is NULL").ok) return;
    staged(c.who, [&](HostCall& hc) {
        auto dw = (const float*)hc.in(w, (size_t)K * N * sizeof(float));
        auto dc = (int8_t*)hc.out(codes, q8_code_bytes(N, K));
        auto ds = (float*)hc.out(scales, q8_scale_bytes(N));
        return !hc.failed() && acfun_dev_quantize_q8(dw, ACFUN_F32, N, K, 1, dc, ds, hc.stream()) == 0;
    });
}

void acfun_fc_q8(const float* input, int N, int Cin, const int8_t* weight, const float* wscale, const float* bias,
                 int Cout, float* output, int act) {
    q8_host_layer({"acfun_fc_q8"}, {N, Cout, Cin, input, nullptr, {weight}, {wscale}, {bias}, output, act, false});
}

void acfun_fc_gated_q8(const float* input, int N, int Cin, const int8_t* gate, const float* gscale,
                       const float* gbias, const int8_t* up, const float* uscale, const float* ubias, int Cout,
                       float* output, int act) {
    q8_host_layer({"acfun_fc_gated_q8"},
                  {N, Cout, Cin, input, nullptr, {gate, up}, {gscale, uscale}, {gbias, ubias}, output, act, true});
}

// ------------------------------------------------------------------ sampling
int acfun_dev_sample(const void* logits, int type, int rows, int cols, int ld, const float* temperature,
                     const int* top_k, const float* top_p, const float* min_p, const float* u, int32_t* token,
                     float* prob, void* stream) {
    Checks c{"acfun_dev_sample"};
    if (!c.type(type).need(rows >= 0 && cols >= 0, "a size is negative").need(ld >= cols, "ld is less than cols").ok)
        return -1;
    if (rows == 0) return 0;
    c.need(cols <= kSampleMaxCols, "more than 2^24 columns").fits(sample_fits(rows));
    if (cols > 0) c.tensor(logits, type, "logits is NULL");
    c.need(u != nullptr, "u is NULL").need(token != nullptr, "token is NULL");
    c.param(temperature).param(top_k).param(top_p).param(min_p).param(u).param(token).param(prob);
    if (!c.ok) return -1;
    const size_t n = cols > 0 ? ((size_t)(rows - 1) * ld + cols) * type_size(type) : 0, np = 4 * (size_t)rows;
    c.apart(token, np, prob, np);
    for (const void* out : {(const void*)token, (const void*)prob}) {
        if (!out) continue;
        c.apart(out, np, logits, n);
        for (const void* in : {(const void*)temperature, (const void*)top_k, (const void*)top_p, (const void*)min_p,
                               (const void*)u})
            c.apart(out, np, in, np);
    }
    if (!c.ok) return -1;
    const SampleArgs a{logits, rows, cols, ld, temperature, top_k, top_p, min_p, u, token, prob};
    return call(c.who, [&] { return sample_rows(a, type, resolve(stream)); });
}

void acfun_sample(const float* logits, int rows, int cols, const float* temperature, const int* top_k,
                  const float* top_p, const float* min_p, const float* u, int32_t* token, float* prob) {
    if (rows <= 0 || cols < 0) return;
    Checks c{"acfun_sample"};
    if (!c.need((cols == 0 || logits) && u && token, "a pointer is NULL").ok) return;
    staged(c.who, [&](HostCall& hc) {
        const size_t n = 4 * (size_t)rows;
        auto dx = (const float*)hc.in(logits, n * cols);
        auto dt = (const float*)hc.in(temperature, n);
        auto dk = (const int*)hc.in(top_k, n);
        auto dp = (const float*)hc.in(top_p, n), dm = (const float*)hc.in(min_p, n), du = (const float*)hc.in(u, n);
        auto to = (int32_t*)hc.out(token, n);
        auto pr = (float*)hc.out(prob, n);
        return !hc.failed() &&
               acfun_dev_sample(dx, ACFUN_F32, rows, cols, cols, dt, dk, dp, dm, du, to, pr, hc.stream()) == 0;
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
