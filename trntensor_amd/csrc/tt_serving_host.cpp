// Host path of the serving operators (part of the tt_fastpath extension).
//
// A decode step makes a few calls of microseconds each, where the checks and
// the argument packing of Python cost more than the kernels. The objects here
// keep what does not change between calls (a matrix's or a cache's pointers
// and sizes) and run a call that has the usual form - operands on the
// matrix's or cache's device, dtypes and shapes that agree, nothing that asks
// for a gradient - with one allocation and one library call on torch's
// current stream. Any other call is declined (None), and the Python front-end
// checks, stages and reports as it always does.
#include <torch/extension.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>
#include <torch/csrc/autograd/forward_grad.h>

#include <cstring>
#include <string>

#include "trntensor_hip.h"

namespace {

using at::Tensor;
using OptTensor = c10::optional<Tensor>;

// Entry points of the loaded libtrntensor_hip.so, by address.
struct Library {
    decltype(&tt_q4_matmul) q4_matmul;
    decltype(&tt_kv_append) kv_append;
    decltype(&tt_kv_attention_workspace_bytes) attention_bytes;
    decltype(&tt_kv_attention) kv_attention;
    decltype(&tt_last_error) last_error;
    decltype(&tt_status_string) status_string;
    decltype(&tt_fp8_quantize) fp8_quantize;
    decltype(&tt_rms_norm) rms_norm;
    decltype(&tt_fp8_matmul) fp8_matmul;
    decltype(&tt_fp8_gated_workspace_bytes) gated_bytes;
    decltype(&tt_fp8_gated_matmul) gated_matmul;

    explicit Library(const std::vector<int64_t>& a) {
        TORCH_CHECK(a.size() == 11, "Library: eleven entry points expected");
        for (int64_t p : a) TORCH_CHECK(p != 0, "Library: null entry point");
        q4_matmul = reinterpret_cast<decltype(q4_matmul)>(a[0]);
        kv_append = reinterpret_cast<decltype(kv_append)>(a[1]);
        attention_bytes = reinterpret_cast<decltype(attention_bytes)>(a[2]);
        kv_attention = reinterpret_cast<decltype(kv_attention)>(a[3]);
        last_error = reinterpret_cast<decltype(last_error)>(a[4]);
        status_string = reinterpret_cast<decltype(status_string)>(a[5]);
        fp8_quantize = reinterpret_cast<decltype(fp8_quantize)>(a[6]);
        rms_norm = reinterpret_cast<decltype(rms_norm)>(a[7]);
        fp8_matmul = reinterpret_cast<decltype(fp8_matmul)>(a[8]);
        gated_bytes = reinterpret_cast<decltype(gated_bytes)>(a[9]);
        gated_matmul = reinterpret_cast<decltype(gated_matmul)>(a[10]);
    }

    void check(int rc, const char* what) const {
        if (rc == TT_OK) return;
        const char* detail = last_error();
        const std::string msg = std::string(what) + ": " + (detail && *detail ? detail : status_string(rc));
        PyErr_SetString(rc == TT_INVALID       ? PyExc_ValueError
                        : rc == TT_UNSUPPORTED ? PyExc_NotImplementedError
                                               : PyExc_RuntimeError,
                        msg.c_str());
        throw py::error_already_set();
    }
};

// Library dtype code of activations, or -1.
int64_t code_of(at::ScalarType t) {
    switch (t) {
        case at::kFloat:
            return TT_F32;
        case at::kBFloat16:
            return TT_BF16;
        case at::kHalf:
            return TT_F16;
        default:
            return -1;
    }
}

struct Place {
    c10::DeviceIndex device;

    // Within forward mode (which no_grad leaves on) operands may have tangents: Python looks for them.
    bool here() const {
        const bool forward =
            c10::AutogradState::get_tls_state().get_fw_grad_mode() && torch::autograd::ForwardADLevel::try_get_by_idx(0);
        return !forward && c10::hip::current_device() == device;
    }
    bool holds(const Tensor& t) const { return t.is_cuda() && t.device().index() == device && !wants_grad(t); }
    static bool wants_grad(const Tensor& t) { return t.requires_grad() && at::GradMode::is_enabled(); }
    Tensor empty(c10::IntArrayRef sizes, at::ScalarType t) const {
        return at::empty(sizes, at::TensorOptions().dtype(t).device(c10::DeviceType::CUDA, device));
    }
    void* stream() const { return c10::hip::getCurrentHIPStream(device).stream(); }
};

class Q4Host {
   public:
    Q4Host(const std::vector<int64_t>& entries, const Tensor& packed, const Tensor& scales, const OptTensor& zeros, int64_t n,
           int64_t k, int64_t group, int64_t scale_code)
        : lib_(entries), packed_(packed), scales_(scales), zeros_(zeros), at_{packed.device().index()} {
        std::memset(&args_, 0, sizeof args_);
        args_.scale_dtype = scale_code;
        args_.N = n;
        args_.K = k;
        args_.group = group;
        args_.ldy = n;
        args_.codes = packed.data_ptr();
        args_.scales = scales.data_ptr();
        args_.zeros = zeros ? zeros->data_ptr() : nullptr;
    }

    py::object run(const Tensor& x) const {
        const int64_t nd = x.dim();
        tt_q4_args a = args_;
        a.dtype = code_of(x.scalar_type());
        if (nd < 1 || a.dtype < 0 || !unmoved() || !at_.holds(x) || !at_.here() || x.size(nd - 1) != a.K) return py::none();
        if (nd == 2 && x.stride(1) == 1 && x.stride(0) >= a.K) {
            a.M = x.size(0);
            a.ldx = x.stride(0);
        } else if (x.is_contiguous()) {
            a.M = x.numel() / a.K;
            a.ldx = a.K;
        } else {
            return py::none();
        }
        c10::SmallVector<int64_t, 5> sizes(x.sizes().begin(), x.sizes().end());
        sizes[nd - 1] = a.N;
        const Tensor y = at_.empty(sizes, x.scalar_type());
        a.x = x.data_ptr();
        a.y = y.data_ptr();
        lib_.check(lib_.q4_matmul(&a, at_.stream()), "tt_q4_matmul");
        return py::cast(y);
    }

   private:
    // The tensors are where they were: else Python reports it.
    bool unmoved() const {
        return packed_.data_ptr() == args_.codes && scales_.data_ptr() == args_.scales &&
               (!zeros_ || zeros_->data_ptr() == args_.zeros);
    }

    Library lib_;
    Tensor packed_, scales_;
    OptTensor zeros_;
    Place at_;
    tt_q4_args args_;
};

class CacheHost {
   public:
    CacheHost(const std::vector<int64_t>& entries, const Tensor& k, const Tensor& v, const Tensor& k_scale, const Tensor& v_scale,
              int64_t dim)
        : lib_(entries), keep_{k, v, k_scale, v_scale}, at_{k.device().index()} {
        cache_.k = k.data_ptr();
        cache_.v = v.data_ptr();
        cache_.k_scale = static_cast<float*>(k_scale.data_ptr());
        cache_.v_scale = static_cast<float*>(v_scale.data_ptr());
        cache_.pages = k.size(0);
        cache_.heads = k.size(1);
        cache_.page = k.size(2);
        cache_.dim = dim;
    }

    // (handled, rotated queries or None)
    py::tuple append(const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& lengths, const OptTensor& counts,
                     const OptTensor& q, const OptTensor& cos, const OptTensor& sin, bool interleaved) const {
        const py::tuple declined = py::make_tuple(false, py::none());
        tt_kv_append_args a;
        std::memset(&a, 0, sizeof a);
        a.dtype = code_of(k.scalar_type());
        if (a.dtype < 0 || k.dim() != 4 || !unmoved() || !at_.here()) return declined;
        a.batch = k.size(0);
        a.tokens = k.size(1);
        if (a.batch < 1 || a.tokens < 1 || !rows(k, a.batch, a.tokens, cache_.heads) || !rows(v, a.batch, a.tokens, cache_.heads) ||
            v.scalar_type() != k.scalar_type() || !schedule(a.batch, table, lengths, counts))
            return declined;
        a.table_width = table.size(1);
        if (cos.has_value() != sin.has_value() || (q && !cos)) return declined;
        if (cos) {
            if (!angles(*cos) || !angles(*sin) || cos->sizes() != sin->sizes()) return declined;
            a.rot = 2 * cos->size(1);
            if (a.rot < 2 || a.rot > cache_.dim || cos->size(0) < a.table_width * cache_.page) return declined;
            a.cos = static_cast<const float*>(cos->data_ptr());
            a.sin = static_cast<const float*>(sin->data_ptr());
        }
        Tensor out;
        if (q) {
            if (q->dim() != 4 || !rows(*q, a.batch, a.tokens, q->size(2)) || q->scalar_type() != k.scalar_type() || q->size(2) < 1)
                return declined;
            a.q_heads = q->size(2);
            out = at_.empty(q->sizes(), q->scalar_type());
            a.q = q->data_ptr();
            a.q_out = out.data_ptr();
            strides(*q, a.q_stride);
        }
        a.interleaved = interleaved;
        a.table_stride = table.stride(0);
        strides(k, a.k_stride);
        strides(v, a.v_stride);
        a.k = k.data_ptr();
        a.v = v.data_ptr();
        a.table = static_cast<const int32_t*>(table.data_ptr());
        a.lengths = static_cast<const int32_t*>(lengths.data_ptr());
        a.counts = counts ? static_cast<const int32_t*>(counts->data_ptr()) : nullptr;
        a.cache = cache_;
        lib_.check(lib_.kv_append(&a, at_.stream()), "tt_kv_append");
        return py::make_tuple(true, q ? py::cast(out) : py::none());
    }

    py::object attention(const Tensor& q, const Tensor& table, const Tensor& lengths, const OptTensor& counts, double scale,
                         int64_t window, int64_t sinks) const {
        tt_kv_attention_args a;
        std::memset(&a, 0, sizeof a);
        a.dtype = code_of(q.scalar_type());
        if (a.dtype < 0 || q.dim() != 4 || !unmoved() || !at_.here() || window < 0 || sinks < 0) return py::none();
        a.batch = q.size(0);
        a.tokens = q.size(1);
        a.q_heads = q.size(2);
        if (a.batch < 1 || a.tokens < 1 || a.q_heads < 1 || a.q_heads % cache_.heads || !rows(q, a.batch, a.tokens, a.q_heads) ||
            !schedule(a.batch, table, lengths, counts))
            return py::none();
        a.window = window;
        a.sinks = sinks;
        a.table_width = table.size(1);
        a.table_stride = table.stride(0);
        strides(q, a.q_stride);
        a.scale = scale;
        const Tensor out = at_.empty(q.sizes(), q.scalar_type());
        a.q = q.data_ptr();
        a.out = out.data_ptr();
        a.table = static_cast<const int32_t*>(table.data_ptr());
        a.lengths = static_cast<const int32_t*>(lengths.data_ptr());
        a.counts = counts ? static_cast<const int32_t*>(counts->data_ptr()) : nullptr;
        a.cache = cache_;
        a.workspace_bytes = static_cast<int64_t>(lib_.attention_bytes(&a));
        Tensor room;
        if (a.workspace_bytes) {
            room = at_.empty({a.workspace_bytes}, at::kByte);
            a.workspace = room.data_ptr();
        }
        lib_.check(lib_.kv_attention(&a, at_.stream()), "tt_kv_attention");
        return py::cast(out);
    }

   private:
    bool unmoved() const {
        return keep_[0].data_ptr() == cache_.k && keep_[1].data_ptr() == cache_.v && keep_[2].data_ptr() == cache_.k_scale &&
               keep_[3].data_ptr() == cache_.v_scale;
    }
    bool rows(const Tensor& t, int64_t batch, int64_t tokens, int64_t heads) const {
        return t.dim() == 4 && t.size(0) == batch && t.size(1) == tokens && t.size(2) == heads && t.size(3) == cache_.dim &&
               (t.stride(3) == 1 || cache_.dim == 1) && at_.holds(t);
    }
    bool schedule(int64_t batch, const Tensor& table, const Tensor& lengths, const OptTensor& counts) const {
        auto list = [&](const Tensor& t) {
            return t.dim() == 1 && t.size(0) == batch && t.scalar_type() == at::kInt && t.is_contiguous() && at_.holds(t);
        };
        return table.dim() == 2 && table.size(0) == batch && table.scalar_type() == at::kInt &&
               (table.stride(1) == 1 || table.size(1) <= 1) && at_.holds(table) && list(lengths) && (!counts || list(*counts));
    }
    bool angles(const Tensor& t) const {
        return t.dim() == 2 && t.scalar_type() == at::kFloat && t.is_contiguous() && at_.holds(t);
    }
    static void strides(const Tensor& t, int64_t* s) {
        for (int i = 0; i < 3; ++i) s[i] = t.stride(i);
    }

    Library lib_;
    Tensor keep_[4];
    Place at_;
    tt_kv_cache cache_;
};

// Codes and scales of rows in 8 bits, as the kernels lay them out.
struct Rows8 {
    Tensor codes, scales;

    Rows8(const Place& at, int64_t rows, int64_t dim) {
        const int64_t blocks = (dim + 127) / 128;
        codes = at.empty({rows, blocks * 128}, at::kFloat8_e4m3fn);
        scales = at.empty({rows, (blocks + 3) / 4 * 4}, at::kFloat8_e8m0fnu);
    }
};

// Rows of `dim` elements of unit stride, `stride` elements apart; false where they are not.
bool rows_of(const Tensor& x, int64_t& rows, int64_t& dim, int64_t& stride) {
    const int64_t nd = x.dim();
    if (nd < 1 || x.size(nd - 1) < 1 || x.is_neg()) return false;
    dim = x.size(nd - 1);
    if (nd == 2 && x.stride(1) == 1) {
        rows = x.size(0);
        stride = x.stride(0);
        return true;
    }
    rows = x.numel() / dim;
    stride = dim;
    return x.is_contiguous();
}

// Norms and quantization.
class RowsHost {
   public:
    explicit RowsHost(const std::vector<int64_t>& entries) : lib_(entries) {}

    // (codes, scales), or None
    py::object quantize(const Tensor& x) const {
        tt_fp8_quantize_args a;
        a.dtype = code_of(x.scalar_type());
        const Place at{x.device().index()};
        if (a.dtype < 0 || !at.holds(x) || !at.here() || !rows_of(x, a.rows, a.dim, a.x_stride)) return py::none();
        const Rows8 out(at, a.rows, a.dim);
        a.x = x.data_ptr();
        a.codes = out.codes.data_ptr();
        a.scales = out.scales.data_ptr();
        lib_.check(lib_.fp8_quantize(&a, at.stream()), "tt_fp8_quantize");
        return py::make_tuple(out.codes, out.scales);
    }

    // (norm or codes, scales or None, sum or None), or None
    py::object norm(const Tensor& x, const OptTensor& weight, const OptTensor& residual, double eps, bool fp8) const {
        tt_rms_norm_args a;
        std::memset(&a, 0, sizeof a);
        a.dtype = code_of(x.scalar_type());
        const Place at{x.device().index()};
        if (a.dtype < 0 || !at.holds(x) || !at.here() || !rows_of(x, a.rows, a.dim, a.x_stride) || !(eps >= 0.0) || eps >= 1e38)
            return py::none();
        if (weight) {
            a.weight_dtype = code_of(weight->scalar_type());
            if (a.weight_dtype < 0 || weight->dim() != 1 || weight->size(0) != a.dim || !weight->is_contiguous() || weight->is_neg() ||
                !at.holds(*weight))
                return py::none();
            a.weight = weight->data_ptr();
        }
        Tensor sum;
        if (residual) {
            int64_t rows, dim;
            if (residual->sizes() != x.sizes() || residual->scalar_type() != x.scalar_type() || !at.holds(*residual) ||
                !rows_of(*residual, rows, dim, a.residual_stride))
                return py::none();
            sum = at.empty(x.sizes(), x.scalar_type());
            a.residual = residual->data_ptr();
            a.sum = sum.data_ptr();
        }
        a.eps = eps;
        a.x = x.data_ptr();
        Tensor first, second;
        if (fp8) {
            const Rows8 out(at, a.rows, a.dim);
            first = out.codes;
            second = out.scales;
            a.codes = first.data_ptr();
            a.scales = second.data_ptr();
        } else {
            first = at.empty(x.sizes(), x.scalar_type());
            a.y = first.data_ptr();
        }
        lib_.check(lib_.rms_norm(&a, at.stream()), "tt_rms_norm");
        return py::make_tuple(first, fp8 ? py::cast(second) : py::none(), residual ? py::cast(sum) : py::none());
    }

   private:
    Library lib_;
};

// 8-bit weights. Rows come as their two arrays and the shape they were made in.
class Fp8Host {
   public:
    Fp8Host(const std::vector<int64_t>& entries, const Tensor& packed, const Tensor& scales, int64_t n, int64_t k, bool e8m0)
        : lib_(entries), packed_(packed), scales_(scales), at_{packed.device().index()}, n_(n), k_(k), code_(e8m0 ? TT_E8M0 : TT_F32) {}

    py::object run(const Tensor& codes, const Tensor& scales, const std::vector<int64_t>& shape, at::ScalarType dtype) const {
        tt_fp8_matmul_args a;
        a.dtype = code_of(dtype);
        if (a.dtype < 0 || !at_.here() || !takes(codes, scales, shape)) return py::none();
        a.scale_dtype = code_;
        a.M = codes.size(0);
        a.N = n_;
        a.K = k_;
        a.x = codes.data_ptr();
        a.x_scales = scales.data_ptr();
        a.w = packed_.data_ptr();
        a.w_scales = scales_.data_ptr();
        const Tensor y = at_.empty(result(shape), dtype);
        a.y = y.data_ptr();
        lib_.check(lib_.fp8_matmul(&a, at_.stream()), "tt_fp8_matmul");
        return py::cast(y);
    }

    // (result or codes, scales or None), or None; this matrix is the gate's.
    py::object gated(const Fp8Host& up, const Tensor& codes, const Tensor& scales, const std::vector<int64_t>& shape,
                     at::ScalarType dtype, int64_t activation, bool fp8) const {
        tt_fp8_gated_args a;
        std::memset(&a, 0, sizeof a);
        a.dtype = code_of(dtype);
        if (a.dtype < 0 || !at_.here() || !takes(codes, scales, shape) || up.n_ != n_ || up.k_ != k_ || up.code_ != code_ ||
            up.at_.device != at_.device)
            return py::none();
        a.scale_dtype = code_;
        a.activation = activation;
        a.M = codes.size(0);
        a.N = n_;
        a.K = k_;
        a.x = codes.data_ptr();
        a.x_scales = scales.data_ptr();
        a.gate = packed_.data_ptr();
        a.gate_scales = scales_.data_ptr();
        a.up = up.packed_.data_ptr();
        a.up_scales = up.scales_.data_ptr();
        Tensor first, second, room;
        if (fp8) {
            const Rows8 out(at_, a.M, n_);
            first = out.codes;
            second = out.scales;
            a.codes = first.data_ptr();
            a.scales = second.data_ptr();
            a.workspace_bytes = static_cast<int64_t>(lib_.gated_bytes(&a));
            if (a.workspace_bytes) {
                room = at_.empty({a.workspace_bytes}, at::kByte);
                a.workspace = room.data_ptr();
            }
        } else {
            first = at_.empty(result(shape), dtype);
            a.y = first.data_ptr();
        }
        lib_.check(lib_.gated_matmul(&a, at_.stream()), "tt_fp8_gated_matmul");
        return py::make_tuple(first, fp8 ? py::cast(second) : py::none());
    }

   private:
    // (Users hold both tensors, and may have resized them.)
    bool takes(const Tensor& codes, const Tensor& scales, const std::vector<int64_t>& shape) const {
        if (shape.empty() || shape.back() != k_ || n_ < 1) return false;
        int64_t count = 1;
        for (size_t i = 0; i + 1 < shape.size(); ++i) count *= shape[i];
        const int64_t blocks = (k_ + 127) / 128;
        return whole(codes, count, blocks * 128) && whole(scales, count, (blocks + 3) / 4 * 4);
    }
    bool whole(const Tensor& t, int64_t rows, int64_t width) const {
        return t.is_cuda() && t.device().index() == at_.device && t.dim() == 2 && t.size(0) == rows && t.size(1) == width &&
               t.is_contiguous() && static_cast<int64_t>(t.storage().nbytes()) >= t.storage_offset() + rows * width;
    }
    std::vector<int64_t> result(std::vector<int64_t> shape) const {
        shape.back() = n_;
        return shape;
    }

    Library lib_;
    Tensor packed_, scales_;
    Place at_;
    int64_t n_, k_, code_;
};

}  // namespace

void bind_serving(py::module_& m) {
    py::class_<Q4Host>(m, "Q4Host")
        .def(py::init<const std::vector<int64_t>&, const Tensor&, const Tensor&, const OptTensor&, int64_t, int64_t, int64_t,
                      int64_t>())
        .def("run", &Q4Host::run);
    py::class_<CacheHost>(m, "CacheHost")
        .def(py::init<const std::vector<int64_t>&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, int64_t>())
        .def("append", &CacheHost::append)
        .def("attention", &CacheHost::attention);
    py::class_<RowsHost>(m, "RowsHost")
        .def(py::init<const std::vector<int64_t>&>())
        .def("quantize", &RowsHost::quantize)
        .def("norm", &RowsHost::norm);
    py::class_<Fp8Host>(m, "Fp8Host")
        .def(py::init<const std::vector<int64_t>&, const Tensor&, const Tensor&, int64_t, int64_t, bool>())
        .def("run", &Fp8Host::run)
        .def("gated", &Fp8Host::gated);
}
