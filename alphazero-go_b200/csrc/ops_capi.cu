// C ABI of the operators beside the network (include/azb200.h): argument
// checks, then one or two launches on the caller's stream. The caller's
// current device is left as it was.
#include <cmath>
#include <stdexcept>
#include <string>

#include "../../include/azb200.h"
#include "capi_types.hpp"
#include "engine.hpp"
#include "ops.hpp"

using namespace azb;

namespace {

// `device` current for the scope.
class OnDevice {
public:
    explicit OnDevice(int device) : info_(&device_info(device)) {
        if (!info_->usable) throw std::runtime_error("cuda: " + info_->why);
        if (cudaGetDevice(&before_) != cudaSuccess) {
            cudaGetLastError();
            before_ = -1;
        }
        if (before_ == device) before_ = -1;   // nothing to put back
        else check(cudaSetDevice(device), "cudaSetDevice");
    }
    ~OnDevice() {
        if (before_ >= 0) cudaSetDevice(before_);
    }
    OnDevice(const OnDevice&) = delete;
    OnDevice& operator=(const OnDevice&) = delete;
    int sms() const { return info_->sms; }

private:
    const DeviceInfo* info_;
    int before_ = -1;
};

void require(bool ok, const std::string& what) {
    if (!ok) throw std::invalid_argument(what);
}

// The largest sizes: a product's tiles are numbered in 32 bits.
constexpr long long kMaxRows = 1ll << 22, kMaxCols = 1ll << 26;

MxShape mx_shape(long long rows, long long cols, const char* fn) {
    require(rows >= 0 && rows <= kMaxRows && cols >= 1 && cols <= kMaxCols,
            std::string(fn) + ": a matrix of " + std::to_string(rows) + " x " + std::to_string(cols) +
                " (rows 0.." + std::to_string(kMaxRows) + ", columns 1.." + std::to_string(kMaxCols) + ")");
    return MxShape{rows, cols};
}

void check_type(int type, const char* fn) {
    require(type == kElemF32 || type == kElemBF16, std::string(fn) + ": unknown element type " + std::to_string(type));
}

void check_ld(long long ld, long long cols, long long rows, const char* fn) {
    require(ld >= 0 && (ld >= cols || rows <= 1), std::string(fn) + ": rows overlap (stride " + std::to_string(ld) + ", " +
                                                      std::to_string(cols) + " columns)");
}

void check_aligned(const void* p, size_t to, const char* what, const char* fn) {
    if (reinterpret_cast<uintptr_t>(p) % to != 0)
        throw std::invalid_argument(std::string(fn) + ": " + what + " must be aligned to " + std::to_string(to) + " bytes");
}

// A quantised operand's two arrays.
void check_mx(const void* codes, const void* scales, const char* what, const char* fn) {
    require(codes && scales, std::string(fn) + ": null " + what);
    check_aligned(codes, 16, what, fn);
    check_aligned(scales, 16, what, fn);
}

cudaStream_t stream_of(void* s) { return static_cast<cudaStream_t>(s); }

size_t round_256(size_t n) { return (n + 255) / 256 * 256; }

}  // namespace

extern "C" {

int azb_mx4_sizes(long long rows, long long cols, size_t* code_bytes, size_t* scale_bytes, char* err, size_t err_cap) {
    return guarded(err, err_cap, "", [&] {
        const MxShape s = mx_shape(rows, cols, "azb_mx4_sizes");
        if (code_bytes) *code_bytes = s.code_bytes();
        if (scale_bytes) *scale_bytes = s.scale_bytes();
    });
}

int azb_mx4_quantise(int device, const void* x, int type, long long rows, long long cols, long long ld, void* codes,
                     void* scales, void* stream, char* err, size_t err_cap) {
    return guarded(err, err_cap, "", [&] {
        const char* fn = "azb_mx4_quantise";
        MxCastArgs a{mx_shape(rows, cols, fn), const_cast<void*>(x), type, ld, static_cast<uint8_t*>(codes),
                     static_cast<uint8_t*>(scales)};
        check_type(type, fn);
        require(ld >= 0, std::string(fn) + ": negative row stride");
        if (rows == 0) return;
        require(x, std::string(fn) + ": null x");
        check_aligned(x, elem_size(type), "x", fn);
        check_mx(codes, scales, "codes or scales", fn);
        const OnDevice on(device);
        check(launch_mx4_quantise(a, on.sms(), stream_of(stream)), fn);
    });
}

int azb_mx4_values(int device, const void* codes, const void* scales, long long rows, long long cols, void* out, int type,
                   long long ld, void* stream, char* err, size_t err_cap) {
    return guarded(err, err_cap, "", [&] {
        const char* fn = "azb_mx4_values";
        MxCastArgs a{mx_shape(rows, cols, fn), out, type, ld, static_cast<uint8_t*>(const_cast<void*>(codes)),
                     static_cast<uint8_t*>(const_cast<void*>(scales))};
        check_type(type, fn);
        check_ld(ld, cols, rows, fn);
        if (rows == 0) return;
        require(out, std::string(fn) + ": null out");
        check_aligned(out, elem_size(type), "out", fn);
        check_mx(codes, scales, "codes or scales", fn);
        const OnDevice on(device);
        check(launch_mx4_values(a, on.sms(), stream_of(stream)), fn);
    });
}

int azb_mx4_product(int device, const void* x_codes, const void* x_scales, long long m, const void* w_codes,
                    const void* w_scales, long long n, long long k, const float* bias, int relu, void* out, int type,
                    long long ld, void* stream, char* err, size_t err_cap) {
    return guarded(err, err_cap, "", [&] {
        const char* fn = "azb_mx4_product";
        mx_shape(m, k, fn);
        mx_shape(n, k, fn);
        check_type(type, fn);
        check_ld(ld, n, m, fn);
        if (m == 0 || n == 0) return;
        require(out, std::string(fn) + ": null out");
        check_aligned(out, elem_size(type), "out", fn);
        check_aligned(bias, 4, "bias", fn);
        check_mx(x_codes, x_scales, "x", fn);
        check_mx(w_codes, w_scales, "w", fn);
        const OnDevice on(device);
        const MxProductArgs a{static_cast<const uint8_t*>(x_codes), static_cast<const uint8_t*>(x_scales),
                              static_cast<const uint8_t*>(w_codes), static_cast<const uint8_t*>(w_scales),
                              m, n, k, bias, relu != 0, out, type, ld, false};
        check(launch_mx4_product(a, on.sms(), stream_of(stream)), fn);
    });
}

size_t azb_mx4_linear_workspace(long long m, long long n, long long k) {
    if (m < 1 || m > kMaxRows || n < 1 || n > kMaxRows || k < 1 || k > kMaxCols || mx4_product_quantises(m, n, k)) return 0;
    const MxShape s{m, k};
    return round_256(s.code_bytes()) + s.scale_bytes();
}

int azb_mx4_linear(int device, const void* x, int x_type, long long m, long long k, long long x_ld, const void* w_codes,
                   const void* w_scales, long long n, const float* bias, int relu, void* out, int type, long long ld,
                   void* workspace, size_t workspace_bytes, void* stream, char* err, size_t err_cap) {
    return guarded(err, err_cap, "", [&] {
        const char* fn = "azb_mx4_linear";
        const MxShape xs = mx_shape(m, k, fn);
        mx_shape(n, k, fn);
        check_type(x_type, fn);
        check_type(type, fn);
        require(x_ld >= 0, std::string(fn) + ": negative row stride");
        check_ld(ld, n, m, fn);
        if (m == 0 || n == 0) return;
        require(x && out, std::string(fn) + ": null x or out");
        check_aligned(x, elem_size(x_type), "x", fn);
        check_aligned(out, elem_size(type), "out", fn);
        check_aligned(bias, 4, "bias", fn);
        check_mx(w_codes, w_scales, "w", fn);
        if (mx4_product_quantises(m, n, k)) {
            const OnDevice on(device);
            const MxProductArgs a{nullptr, nullptr, static_cast<const uint8_t*>(w_codes), static_cast<const uint8_t*>(w_scales),
                                  m, n, k, bias, relu != 0, out, type, ld, false, x, x_type, x_ld};
            check(launch_mx4_product(a, on.sms(), stream_of(stream)), fn);
            return;
        }
        const size_t need = azb_mx4_linear_workspace(m, n, k);
        require(workspace && workspace_bytes >= need,
                std::string(fn) + ": the workspace holds " + std::to_string(workspace_bytes) + " bytes of " + std::to_string(need));
        check_aligned(workspace, 256, "the workspace", fn);
        uint8_t* codes = static_cast<uint8_t*>(workspace);
        uint8_t* scales = codes + round_256(xs.code_bytes());
        const OnDevice on(device);
        const MxCastArgs q{xs, const_cast<void*>(x), x_type, x_ld, codes, scales};
        check(launch_mx4_quantise(q, on.sms(), stream_of(stream)), fn);
        const MxProductArgs a{codes, scales, static_cast<const uint8_t*>(w_codes), static_cast<const uint8_t*>(w_scales),
                              m, n, k, bias, relu != 0, out, type, ld, true};
        check(launch_mx4_product(a, on.sms(), stream_of(stream)), fn);
    });
}

int azb_sample_moves(int device, const azb_sample_args* p, void* stream, char* err, size_t err_cap) {
    return guarded(err, err_cap, "", [&] {
        const char* fn = "azb_sample_moves";
        require(p, std::string(fn) + ": null argument");
        check_type(p->type, fn);
        require(p->rows >= 0 && p->rows <= (1ll << 27) && p->cols >= 1 && p->cols <= (1ll << 30),
                std::string(fn) + ": " + std::to_string(p->rows) + " rows of " + std::to_string(p->cols) +
                    " (rows 0..2^27, columns 1..2^30)");
        require(p->ld >= 0 && p->noise_ld >= 0 && p->legal_ld >= 0, std::string(fn) + ": negative row stride");
        require(p->temperature_rows || (p->temperature >= 0.0f && std::isfinite(p->temperature)),
                std::string(fn) + ": the temperature must be finite and at least 0");
        require(p->top_k_rows || p->top_k >= 0, std::string(fn) + ": top_k must be at least 0 (0: off)");
        require(p->top_p_rows || (p->top_p >= 0.0f && p->top_p <= 1.0f), std::string(fn) + ": top_p must be in [0, 1]");
        require(p->min_p_rows || (p->min_p >= 0.0f && p->min_p <= 1.0f), std::string(fn) + ": min_p must be in [0, 1]");
        if (p->rows == 0) return;
        require(p->logits && p->moves, std::string(fn) + ": null logits or moves");
        require(p->noise || (!p->temperature_rows && p->temperature == 0.0f),
                std::string(fn) + ": null noise (only temperature 0 needs none)");
        check_aligned(p->logits, elem_size(p->type), "logits", fn);
        check_aligned(p->noise, 4, "noise", fn);
        check_aligned(p->moves, 8, "moves", fn);
        check_aligned(p->logprob, 4, "logprob", fn);
        check_aligned(p->temperature_rows, 4, "temperature_rows", fn);
        check_aligned(p->top_p_rows, 4, "top_p_rows", fn);
        check_aligned(p->min_p_rows, 4, "min_p_rows", fn);
        check_aligned(p->top_k_rows, 4, "top_k_rows", fn);
        const SampleArgs a{p->logits, p->type, p->rows, p->ld, int(p->cols), p->noise, p->noise_ld, p->legal, p->legal_ld,
                           p->temperature, p->top_p, p->min_p, p->top_k, p->temperature_rows, p->top_p_rows,
                           p->min_p_rows, p->top_k_rows, reinterpret_cast<long long*>(p->moves), p->logprob};
        const OnDevice on(device);
        check(launch_sample_moves(a, stream_of(stream)), fn);
    });
}

int azb_ops_check(int device, char* err, size_t err_cap) {
    return guarded(err, err_cap, "", [&] {
        const OnDevice on(device);
        int code = 0;
        check(mx4_error(&code), "azb_ops_check");
        if (code) throw std::runtime_error("cuda: " + kernel_error_text(code));
    });
}

int azb_probe_ops_wait(int device, unsigned long long limit_ns, char* err, size_t err_cap) {
    return guarded(err, err_cap, "", [&] {
        const OnDevice on(device);
        check(mx4_error_probe(limit_ns), "azb_probe_ops_wait");
    });
}

const float* azb_infer_device_logits(azb_infer* h) { return h ? h->impl->device_logits() : nullptr; }

}  // extern "C"
