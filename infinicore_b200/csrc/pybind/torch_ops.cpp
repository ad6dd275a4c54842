// _torch_ops: the operators over quantised pools on torch tensors, for calls whose own time on the GPU is a few microseconds.
//
// What ops.py does in Python for the other operators is done here in C++: the checks of devices, the key of the
// descriptor cache (the cache of include/infinicore_b200/ops.hpp: one for each thread and device, least recently used
// evicted), the current stream, the call through the C ABI.  Scratch comes from torch's caching allocator for each call and
// is reused in the order of the stream.  While a stream is being captured into a CUDA graph, by torch.cuda.graph or by any other
// means, its calls share one scratch buffer that stays allocated for as long as the graph, or one instantiated from it, lives: graphs may
// be replayed at the same time, and beside anything else that torch allocates.
#include <torch/csrc/utils/pybind.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include "infinicore_b200/ops.hpp"

#include <cuda_runtime_api.h>

#include <array>
#include <atomic>
#include <memory>
#include <mutex>
#include <optional>
#include <string>
#include <tuple>
#include <vector>

namespace py = pybind11;
namespace ib = infinicore_b200;

namespace {

infiniDtype_t dtypeOf(const at::Tensor &t) {
    switch (t.scalar_type()) {
    case at::kHalf:
        return INFINI_DTYPE_F16;
    case at::kBFloat16:
        return INFINI_DTYPE_BF16;
    case at::kFloat:
        return INFINI_DTYPE_F32;
    case at::kDouble:
        return INFINI_DTYPE_F64;
    case at::kChar:
        return INFINI_DTYPE_I8;
    case at::kByte:
        return INFINI_DTYPE_U8;
    case at::kShort:
        return INFINI_DTYPE_I16;
    case at::kInt:
        return INFINI_DTYPE_I32;
    case at::kLong:
        return INFINI_DTYPE_I64;
    case at::kBool:
        return INFINI_DTYPE_BOOL;
    default:
        return INFINI_DTYPE_INVALID; // refused with the status of a wrong dtype
    }
}

// A tensor descriptor for the creation of an operator descriptor; none for a tensor that is left out.
class Described {
public:
    explicit Described(const at::Tensor *t) {
        if (t != nullptr) {
            const std::vector<size_t> shape(t->sizes().begin(), t->sizes().end());
            const std::vector<ptrdiff_t> strides(t->strides().begin(), t->strides().end());
            ib::check(infiniopCreateTensorDescriptor(&desc_, shape.size(), shape.data(), strides.data(), dtypeOf(*t)),
                      "infiniopCreateTensorDescriptor");
        }
    }
    Described(const Described &) = delete;
    Described &operator=(const Described &) = delete;
    ~Described() {
        if (desc_ != nullptr) {
            infiniopDestroyTensorDescriptor(desc_);
        }
    }
    infiniopTensorDescriptor_t get() const { return desc_; }

private:
    infiniopTensorDescriptor_t desc_ = nullptr;
};

// The device of all tensors (null: left out), or what is wrong with them.
int deviceOf(const at::Tensor *const *tensors, size_t n) {
    int device = -1;
    for (size_t i = 0; i < n; ++i) {
        if (tensors[i] == nullptr) {
            continue;
        }
        if (!tensors[i]->is_cuda()) {
            throw std::runtime_error("infinicore_b200 operators run on CUDA tensors only; there is no CPU fallback");
        }
        const int here = tensors[i]->get_device();
        if (device >= 0 && here != device) {
            throw std::runtime_error("all tensors of one call must live on the same GPU");
        }
        device = here;
    }
    return device;
}

// Key of the descriptor cache: the operator and everything of its tensors that a descriptor depends on.
const std::string &keyOf(const char *op, const at::Tensor *const *tensors, size_t n, float scale) {
    thread_local std::string key;
    key.assign(op);
    key.push_back('\0');
    auto raw = [&](const void *p, size_t bytes) { key.append(static_cast<const char *>(p), bytes); };
    raw(&scale, sizeof(scale));
    for (size_t i = 0; i < n; ++i) {
        if (tensors[i] == nullptr) {
            key.push_back('-');
            continue;
        }
        const at::Tensor &t = *tensors[i];
        key.push_back(static_cast<char>(t.scalar_type()));
        key.push_back(static_cast<char>(t.dim()));
        raw(t.sizes().data(), sizeof(int64_t) * t.dim());
        raw(t.strides().data(), sizeof(int64_t) * t.dim());
    }
    return key;
}

struct Call {
    Call(const at::Tensor *const *tensors, size_t n) : device(deviceOf(tensors, n)), guard(static_cast<c10::DeviceIndex>(device)) {
        infiniDevice_t kind = INFINI_DEVICE_CPU;
        int id = -1;
        ib::check(infinirtGetDevice(&kind, &id), "infinirtGetDevice");
        if (kind != INFINI_DEVICE_NVIDIA || id != device) { // the handle of a thread is its current infinirt device's
            ib::check(infinirtSetDevice(INFINI_DEVICE_NVIDIA, device), "infinirtSetDevice");
        }
        stream = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream();
    }
    int device;
    c10::cuda::CUDAGuard guard;
    void *stream = nullptr;
};

template <size_t N, typename Create>
const ib::detail::Entry &lookup(const char *op, const std::array<const at::Tensor *, N> &tensors, float scale, Create create,
                                infiniStatus_t (*workspace)(InfiniopDescriptor *, size_t *), infiniStatus_t (*destroy)(InfiniopDescriptor *),
                                const char *what) {
    ib::detail::DeviceState &st = ib::detail::state();
    const std::string &key = keyOf(op, tensors.data(), N, scale);
    if (const ib::detail::Entry *hit = st.cache.get(key)) {
        return *hit;
    }
    ib::detail::Entry e;
    e.destroy = destroy;
    {
        std::vector<std::unique_ptr<Described>> descs;
        std::array<infiniopTensorDescriptor_t, N> d;
        for (size_t i = 0; i < N; ++i) {
            descs.push_back(std::make_unique<Described>(tensors[i]));
            d[i] = descs.back()->get();
        }
        ib::check(create(st.handle, &e.desc, d), what);
    }
    const infiniStatus_t status = workspace(e.desc, &e.workspace_bytes);
    if (status != INFINI_STATUS_SUCCESS) {
        destroy(e.desc);
        throw ib::StatusError(status, what);
    }
    return *st.cache.put(key, e);
}

// Scratch buffers whose graphs are gone.  A graph's last reference is dropped by the CUDA driver, on a thread of its own and where no CUDA
// call may be made: the buffer goes to this list, and back to the allocator at a later call.
struct Released {
    std::mutex mutex;
    std::vector<at::Tensor> tensors;
    std::atomic<bool> any{false};
};
Released &released() {
    static Released *r = new Released; // never destroyed: graphs may outlive static objects
    return *r;
}
void CUDART_CB releaseScratch(void *tensor) {
    Released &r = released();
    const std::lock_guard<std::mutex> lock(r.mutex);
    r.tensors.push_back(*static_cast<at::Tensor *>(tensor));
    delete static_cast<at::Tensor *>(tensor);
    r.any = true;
}

// The buffer of the calls that are being captured on a stream.
struct Captured {
    unsigned long long id = 0; // of the capture; unique in the process
    void *stream = nullptr;
    at::Tensor tensor;
};

void checkCuda(cudaError_t e, const char *what) {
    if (e != cudaSuccess) {
        (void)cudaGetLastError();
        throw std::runtime_error(std::string(what) + ": " + cudaGetErrorString(e));
    }
}

at::Tensor scratch(const at::Tensor &like, size_t bytes, void *stream) {
    thread_local std::vector<Captured> captures;
    const auto fresh = [&] { return at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte)); };
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    unsigned long long id = 0;
    cudaGraph_t graph = nullptr;
    if (cudaStreamGetCaptureInfo(static_cast<cudaStream_t>(stream), &status, &id, &graph) != cudaSuccess) {
        (void)cudaGetLastError(); // the legacy stream while another one is captured: the launch will say so
        return fresh();
    }
    if (status != cudaStreamCaptureStatusActive) {
        captures.clear(); // their graphs hold them
        Released &r = released();
        if (r.any) {
            std::vector<at::Tensor> gone;
            {
                const std::lock_guard<std::mutex> lock(r.mutex);
                gone.swap(r.tensors);
                r.any = false;
            }
        }
        return fresh();
    }
    size_t kept = 0;
    for (size_t i = 0; i < captures.size(); ++i) { // of earlier captures, what is left is their graphs' business
        if (captures[i].id == id) {
            std::swap(captures[kept++], captures[i]);
        }
    }
    captures.resize(kept);
    for (const Captured &c : captures) {
        if (c.stream == stream && c.tensor.numel() >= static_cast<int64_t>(bytes)) {
            return c.tensor;
        }
    }
    auto held = std::make_unique<at::Tensor>(fresh());
    const at::Tensor tensor = *held;
    cudaUserObject_t owner = nullptr;
    checkCuda(cudaUserObjectCreate(&owner, held.get(), releaseScratch, 1, cudaUserObjectNoDestructorSync), "cudaUserObjectCreate");
    (void)held.release();
    const cudaError_t e = cudaGraphRetainUserObject(graph, owner, 1, cudaGraphUserObjectMove);
    if (e != cudaSuccess) {
        (void)cudaUserObjectRelease(owner, 1);
        checkCuda(e, "cudaGraphRetainUserObject");
    }
    captures.push_back({id, stream, tensor});
    return tensor;
}

void quantPagedCaching(const at::Tensor &k_cache, const at::Tensor &v_cache, const at::Tensor &k_scales, const at::Tensor &v_scales,
                       const at::Tensor &k, const at::Tensor &v, const at::Tensor &slot_mapping) {
    const std::array<const at::Tensor *, 7> t = {&k_cache, &v_cache, &k_scales, &v_scales, &k, &v, &slot_mapping};
    const Call call(t.data(), t.size());
    const ib::detail::Entry &e = lookup(
        "torch quant_paged_caching", t, 0.f,
        [](infiniopHandle_t h, InfiniopDescriptor **out, const std::array<infiniopTensorDescriptor_t, 7> &d) {
            return infiniopCreateQuantPagedCachingDescriptor(h, out, d[0], d[1], d[2], d[3], d[4], d[5], d[6]);
        },
        infiniopGetQuantPagedCachingWorkspaceSize, infiniopDestroyQuantPagedCachingDescriptor, "infiniopCreateQuantPagedCachingDescriptor");
    ib::check(infiniopQuantPagedCaching(e.desc, nullptr, 0, k_cache.data_ptr(), v_cache.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr(),
                                        k.data_ptr(), v.data_ptr(), slot_mapping.data_ptr(), call.stream),
              "infiniopQuantPagedCaching");
}

void quantPagedCacheRead(const at::Tensor &k, const at::Tensor &v, const at::Tensor &k_cache, const at::Tensor &v_cache,
                         const at::Tensor &k_scales, const at::Tensor &v_scales, const at::Tensor &slot_mapping) {
    const std::array<const at::Tensor *, 7> t = {&k, &v, &k_cache, &v_cache, &k_scales, &v_scales, &slot_mapping};
    const Call call(t.data(), t.size());
    const ib::detail::Entry &e = lookup(
        "torch quant_paged_cache_read", t, 0.f,
        [](infiniopHandle_t h, InfiniopDescriptor **out, const std::array<infiniopTensorDescriptor_t, 7> &d) {
            return infiniopCreateQuantPagedCacheReadDescriptor(h, out, d[0], d[1], d[2], d[3], d[4], d[5], d[6]);
        },
        infiniopGetQuantPagedCacheReadWorkspaceSize, infiniopDestroyQuantPagedCacheReadDescriptor,
        "infiniopCreateQuantPagedCacheReadDescriptor");
    ib::check(infiniopQuantPagedCacheRead(e.desc, nullptr, 0, k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                                          k_scales.data_ptr(), v_scales.data_ptr(), slot_mapping.data_ptr(), call.stream),
              "infiniopQuantPagedCacheRead");
}

// The same into new rows of `dtype`.
std::tuple<at::Tensor, at::Tensor> quantPagedCacheReadNew(const at::Tensor &k_cache, const at::Tensor &v_cache, const at::Tensor &k_scales,
                                                          const at::Tensor &v_scales, const at::Tensor &slot_mapping, at::ScalarType dtype) {
    if (k_cache.dim() != 4 || v_cache.dim() != 4 || slot_mapping.dim() != 1) {
        throw ib::StatusError(INFINI_STATUS_BAD_TENSOR_SHAPE, "quant_paged_cache_read");
    }
    const std::array<const at::Tensor *, 5> t = {&k_cache, &v_cache, &k_scales, &v_scales, &slot_mapping};
    deviceOf(t.data(), t.size());
    const int64_t packed = k_cache.scalar_type() == at::kByte ? 2 : 1;
    auto rows = [&](const at::Tensor &c) {
        return at::empty({slot_mapping.size(0), c.size(1), c.size(3) * packed}, c.options().dtype(dtype));
    };
    at::Tensor k = rows(k_cache), v = rows(v_cache);
    quantPagedCacheRead(k, v, k_cache, v_cache, k_scales, v_scales, slot_mapping);
    return {k, v};
}

void quantPagedAttention(const at::Tensor &out, const at::Tensor &q, const at::Tensor &k_cache, const at::Tensor &v_cache,
                         const at::Tensor &k_scales, const at::Tensor &v_scales, const at::Tensor &block_tables, const at::Tensor &cache_lens,
                         const std::optional<at::Tensor> &alibi_slopes, double scale_) {
    const float scale = static_cast<float>(scale_);
    const at::Tensor *alibi = alibi_slopes.has_value() ? &*alibi_slopes : nullptr;
    const std::array<const at::Tensor *, 9> t = {&out, &q, &k_cache, &v_cache, &k_scales, &v_scales, &block_tables, &cache_lens, alibi};
    const Call call(t.data(), t.size());
    const ib::detail::Entry &e = lookup(
        "torch quant_paged_attention", t, scale,
        [scale](infiniopHandle_t h, InfiniopDescriptor **o, const std::array<infiniopTensorDescriptor_t, 9> &d) {
            return infiniopCreateQuantPagedAttentionDescriptor(h, o, d[0], d[1], d[2], d[3], d[4], d[5], d[6], d[7], d[8], scale);
        },
        infiniopGetQuantPagedAttentionWorkspaceSize, infiniopDestroyQuantPagedAttentionDescriptor,
        "infiniopCreateQuantPagedAttentionDescriptor");
    at::Tensor workspace; // back to the allocator on return, unless a graph holds it: reused behind this call on its stream
    if (e.workspace_bytes > 0) {
        workspace = scratch(q, e.workspace_bytes, call.stream);
    }
    ib::check(infiniopQuantPagedAttention(e.desc, e.workspace_bytes > 0 ? workspace.data_ptr() : nullptr, e.workspace_bytes, out.data_ptr(),
                                          q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr(),
                                          block_tables.data_ptr(), cache_lens.data_ptr(), alibi != nullptr ? alibi->data_ptr() : nullptr,
                                          call.stream),
              "infiniopQuantPagedAttention");
}

} // namespace

PYBIND11_MODULE(_torch_ops, m) {
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) {
                std::rethrow_exception(p);
            }
        } catch (const ib::StatusError &e) {
            py::object type = py::module_::import("infinicore_b200.libinfiniop").attr("InfiniStatusError");
            PyErr_SetObject(type.ptr(), type(static_cast<int>(e.status)).ptr());
        }
    });
    m.def("quant_paged_caching", &quantPagedCaching);
    m.def("quant_paged_cache_read", &quantPagedCacheRead);
    m.def("quant_paged_cache_read_new", &quantPagedCacheReadNew);
    m.def("quant_paged_attention", &quantPagedAttention);
    // destroys the calling thread's cached descriptors for its current device
    m.def("clear_cache", [] { ib::clear_cache(); });
}
