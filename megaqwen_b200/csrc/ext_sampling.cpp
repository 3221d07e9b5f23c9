// Torch binding of mq_sample (include/megaqwen_b200.h, "sampling"): argument
// checks that raise RuntimeError, the output from the caching allocator on the
// current stream.  The Python name is in megaqwen_b200/sampling.py.

#include <torch/extension.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <cmath>
#include <stdexcept>
#include <string>

#include "megaqwen_b200.h"

namespace {

using torch::Tensor;

[[noreturn]] void fail(const std::string& what) { throw std::runtime_error(what); }

// A parameter: a number for all rows, or a contiguous tensor with one for each.
template <typename T>
const T* per_row(const py::object& x, const Tensor& logits, const char* name, torch::ScalarType type, T* value) {
    if (THPVariable_Check(x.ptr())) {
        const Tensor& t = THPVariable_Unpack(x.ptr());
        if (t.device() != logits.device()) fail(std::string(name) + " must be on " + logits.device().str());
        if (t.scalar_type() != type || t.dim() != 1 || !t.is_contiguous() || t.size(0) != logits.size(0))
            fail(std::string(name) + " must be a contiguous " + (type == torch::kInt32 ? "int32" : "float32") + " tensor with one entry per row");
        return t.data_ptr<T>();
    }
    const double v = PyFloat_AsDouble(x.ptr());
    if (PyErr_Occurred()) {
        PyErr_Clear();
        fail(std::string(name) + " must be a number or a tensor");
    }
    if (!(v >= -2147483648.0 && v <= 3.4e38) || (type == torch::kInt32 && (v > 2147483647.0 || v != std::floor(v))))
        fail(std::string(name) + " is out of range");
    *value = (T)v;
    return nullptr;
}

Tensor sample(Tensor logits, Tensor u, py::object temperature, py::object top_k, py::object top_p, py::object min_p) {
    if (!logits.is_cuda()) fail("logits must be a CUDA tensor");
    mq_sample_params p = {};
    switch (logits.scalar_type()) {
        case torch::kFloat32: p.dtype = MQ_FP32; break;
        case torch::kBFloat16: p.dtype = MQ_BF16; break;
        case torch::kHalf: p.dtype = MQ_FP16; break;
        default: fail("logits must be float32, bfloat16 or float16");
    }
    if (logits.dim() != 2 || logits.size(1) < 1 || logits.size(1) > (1 << 20) || logits.size(0) > (1 << 24))
        fail("logits must be [rows, vocab] with a vocab of 1 to 2^20 and at most 2^24 rows");
    const auto dev = logits.device();
    if (u.device() != dev) fail("u must be on " + dev.str());
    if (u.scalar_type() != torch::kFloat32 || u.dim() != 1 || !u.is_contiguous() || u.size(0) != logits.size(0))
        fail("u must be a contiguous float32 tensor with one entry per row");
    p.temperatures = per_row<float>(temperature, logits, "temperature", torch::kFloat32, &p.temperature);
    p.top_ks = per_row<int>(top_k, logits, "top_k", torch::kInt32, &p.top_k);
    p.top_ps = per_row<float>(top_p, logits, "top_p", torch::kFloat32, &p.top_p);
    p.min_ps = per_row<float>(min_p, logits, "min_p", torch::kFloat32, &p.min_p);
    if (!p.temperatures && p.temperature < 0.f) fail("temperature must not be negative");
    if (!p.top_ps && (p.top_p < 0.f || p.top_p > 1.f)) fail("top_p must be between 0 and 1");
    if (!p.min_ps && (p.min_p < 0.f || p.min_p > 1.f)) fail("min_p must be between 0 and 1");
    c10::cuda::CUDAGuard guard(dev);
    Tensor x = logits;
    if (x.size(1) > 1 && x.stride(1) != 1) x = x.contiguous();
    Tensor out(at::detail::empty_cuda({x.size(0)}, torch::kInt32, dev, c10::nullopt));
    p.logits = x.data_ptr();
    p.row_stride = x.stride(0);
    p.n = (int)x.size(0);
    p.vocab = (int)x.size(1);
    p.u = u.data_ptr<float>();
    p.tokens = out.data_ptr<int>();
    const int rc = mq_sample(&p, c10::cuda::getCurrentCUDAStream(dev.index()).stream());
    if (rc)
        fail(std::string("sample: ") + mq_error_string(rc) + " (code " + std::to_string(rc) + ")" +
             (rc == MQ_ERR_CUDA ? std::string(" ") + mq_last_error_detail() : ""));
    return out;
}

}  // namespace

void bind_sampling(py::module_& m) {
    m.def("sample", &sample, py::arg("logits"), py::arg("u"), py::arg("temperature") = 1.0, py::arg("top_k") = 0,
          py::arg("top_p") = 1.0, py::arg("min_p") = 0.0);
}
