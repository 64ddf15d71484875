// Host side of one QuantLinear.forward call in native code.
//
// A decode GEMV runs for 3..10 us on the device; preparing its launch from Python (attribute look-ups, argument
// conversion of a ctypes call, torch.empty) took 12..16 us per call and the GEMM's 27..31 us, so a loop of small calls
// was bound by the host.  This module does the same checks and the same library call from C++: `Layer.run(x,
// module.__dict__)` returns the output tensor, or None when anything about the call is not the prepared case (another
// device, other buffers, a row count without a plan, a tensor subclass); the caller then takes the Python route,
// which prepares what is missing.  Nothing here launches kernels of its own: the work goes through the C ABI.
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/AutogradState.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <string>
#include <unordered_map>
#include <utility>

#include "../../../../include/b200gptq.h"

namespace {

constexpr int kMaxGemvRows = 16;

// Scratch buffers by (device, stream), registered by ops.get_workspace.  Read and written under the GIL; `owner` is the
// tensor, held while it is registered and by a call that works without the GIL.  in_graph: it was handed out while its stream
// was being captured, so a graph may hold its address for good.
struct Scratch { PyObject* owner; void* ptr; size_t bytes; bool in_graph; };
struct KeyHash {
    size_t operator()(const std::pair<int, void*>& k) const {
        return std::hash<void*>()(k.second) * 31u + (size_t)k.first;
    }
};
std::unordered_map<std::pair<int, void*>, Scratch, KeyHash>* g_scratch;
PyObject* g_get_workspace;   // ops.get_workspace, for a stream without a large enough buffer

PyObject *s_buffers, *s_qweight, *s_g_idx, *s_qzeros, *s_scales, *s_bias, *s_gemv_tuning;

struct GemvEntry {
    PyObject* owner;      // the ops.GemvPlan that owns the handle
    const b200gptq_gemv_plan* plan;
    size_t need;
};

struct Layer {
    PyObject_HEAD
    int K, N, bits, group_size, device;
    // the buffers this object was prepared for: addresses of qweight / g_idx, identity and addresses of the others, and how
    // often the weights, scales and zero-points had been written to
    const void *qweight_at, *g_idx_at;
    uint32_t writes;
    PyObject *qzeros, *scales, *bias, *tuning;
    GemvEntry gemv[kMaxGemvRows + 1];
    // run-time layout for the GEMM (gemm_ok false: no tensor-core kernel for this layer)
    bool gemm_ok;
    int gemv_rows;        // largest row count that goes through plans (8, or 16 where the streaming kernel takes the layer)
    const int32_t *qweight_run, *qzeros_run, *g_idx_run, *x_perm;
    const void *scales_run, *bias_run;
    PyObject* keep;       // keeps the tensors behind those addresses alive
};

// A reference held for the time of a call.
struct Held {
    PyObject* o;
    explicit Held(PyObject* p, bool own = false) : o(p) { if (!own) Py_XINCREF(o); }      // own: a reference that is handed over
    ~Held() { Py_XDECREF(o); }
    Held(const Held&) = delete;
    Held& operator=(const Held&) = delete;
};
// The GIL given up for the time of a scope.
struct WithoutGil {
    PyThreadState* state = PyEval_SaveThread();
    ~WithoutGil() { PyEval_RestoreThread(state); }
};

// Tensors that stand for something else: wrappers without memory of their own (vmap, grad and their kin), views whose values
// are not what lies in memory.
const c10::DispatchKeySet kNotPlain({c10::DispatchKey::Python, c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::BatchedNestedTensor,
                                     c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Functionalize, c10::DispatchKey::Conjugate,
                                     c10::DispatchKey::Negative, c10::DispatchKey::ZeroTensor});

inline const void* tensor_address(PyObject* t) {
    return t && t != Py_None && THPVariable_Check(t) ? THPVariable_Unpack(t).unsafeGetTensorImpl()->data() : nullptr;
}
// Writes in place to a tensor so far (tensors of inference mode do not count them).
inline uint32_t writes_to(PyObject* t) {
    c10::TensorImpl* impl = THPVariable_Unpack(t).unsafeGetTensorImpl();
    return impl->is_inference() ? 0u : impl->version_counter().current_version();
}
inline bool lies_at(PyObject* t, const void* at) {
    return t && THPVariable_Check(t) && THPVariable_Unpack(t).unsafeGetTensorImpl()->data() == at;
}

// (the legacy default stream cannot be captured)
bool is_capturing(cudaStream_t stream) {
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    if (stream) C10_CUDA_CHECK(cudaStreamIsCapturing(stream, &status));
    return status != cudaStreamCaptureStatusNone;
}

bool scratch_for(int device, cudaStream_t stream, size_t need, Scratch* out) {
    auto it = g_scratch->find({device, (void*)stream});
    if (it != g_scratch->end() && !it->second.in_graph) it->second.in_graph = is_capturing(stream);
    if (it == g_scratch->end() || it->second.bytes < need) {
        PyObject* r = PyObject_CallFunction(g_get_workspace, "in", device, (Py_ssize_t)need);
        if (!r) return false;
        Py_DECREF(r);
        it = g_scratch->find({device, (void*)stream});
        if (it == g_scratch->end() || it->second.bytes < need) {
            PyErr_SetString(PyExc_RuntimeError, "no scratch buffer was registered for this stream");
            return false;
        }
    }
    *out = it->second;
    return true;
}

// The module's forward, or None where the prepared case does not apply.
PyObject* run_prepared(Layer* self, PyObject* px, PyObject* dict) {
    if (!THPVariable_CheckExact(px) || !PyDict_Check(dict)) Py_RETURN_NONE;
    const at::Tensor& x = THPVariable_Unpack(px);
    if (x.key_set().has_any(kNotPlain)) Py_RETURN_NONE;
    const int64_t dims = x.dim();
    if (!x.is_cuda() || x.scalar_type() != at::kHalf || dims < 1 || x.size(-1) != self->K || !x.is_contiguous() ||
        x.get_device() != self->device)
        Py_RETURN_NONE;
    const int64_t M = x.numel() / self->K;
    if (M < 1) Py_RETURN_NONE;
    // the module's buffers are the ones this object was prepared for
    PyObject* buffers = PyDict_GetItem(dict, s_buffers);
    if (!buffers) Py_RETURN_NONE;
    PyObject *qweight = PyDict_GetItem(buffers, s_qweight), *g_idx = PyDict_GetItem(buffers, s_g_idx);
    if (!lies_at(qweight, self->qweight_at) || !lies_at(g_idx, self->g_idx_at)) Py_RETURN_NONE;
    PyObject* bias = PyDict_GetItem(buffers, s_bias);
    if (!bias) bias = PyDict_GetItem(dict, s_bias);
    if ((bias ? bias : Py_None) != self->bias || PyDict_GetItem(buffers, s_qzeros) != self->qzeros ||
        PyDict_GetItem(buffers, s_scales) != self->scales)
        Py_RETURN_NONE;
    // (`tensor.data = other` keeps the tensor and moves its numbers)
    auto at = [](PyObject* t) { return THPVariable_Unpack(t).unsafeGetTensorImpl()->data(); };
    if (at(self->qzeros) != self->qzeros_run || at(self->scales) != self->scales_run ||
        (self->bias_run && at(self->bias) != self->bias_run))
        Py_RETURN_NONE;
    // (weights that have been written to: the Python route re-orders them anew, or sees to it that they can be read early)
    if (writes_to(qweight) + writes_to(g_idx) + writes_to(self->qzeros) + writes_to(self->scales) != self->writes) Py_RETURN_NONE;
    const bool gemv = M <= self->gemv_rows;
    const GemvEntry* e = gemv ? &self->gemv[M] : nullptr;
    if (gemv ? (!e->plan || PyDict_GetItem(dict, s_gemv_tuning) != self->tuning) : !self->gemm_ok) Py_RETURN_NONE;
    if (c10::cuda::current_device() != self->device || M > INT32_MAX) Py_RETURN_NONE;

    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)self->device).stream();
    Scratch ws;
    const size_t need = gemv ? e->need : b200gptq_workspace_bytes(B200GPTQ_OP_GEMM, (int)M, self->K, self->N, self->bits);
    if (!scratch_for(self->device, stream, need, &ws)) return nullptr;
    // What another thread may replace while this one has given up the GIL.  (`self`, its tensors and x are held by the caller.)
    const b200gptq_gemv_plan* plan = gemv ? e->plan : nullptr;
    const Held scratch(ws.owner), owner(gemv ? e->owner : nullptr);
    c10::SmallVector<int64_t, 4> shape(x.sizes().begin(), x.sizes().end());
    shape.back() = self->N;
    at::Tensor y;
    int st;
    {
        // A launch waits while the device's queue is full, an allocation may wait for the device: other threads go on.
        const WithoutGil released;
        y = at::detail::empty_cuda(shape, at::kHalf, at::Device(at::kCUDA, (c10::DeviceIndex)self->device), std::nullopt);
        const void* xp = x.unsafeGetTensorImpl()->data();
        void* yp = y.unsafeGetTensorImpl()->mutable_data();
        if (gemv)
            st = b200gptq_gemv_plan_run(plan, xp, yp, ws.ptr, ws.bytes, stream);
        else
            st = b200gptq_gemm(xp, self->qweight_run, self->qzeros_run, self->scales_run, self->g_idx_run, self->x_perm,
                               self->bias_run, yp, (int)M, self->K, self->N, self->bits, self->group_size, ws.ptr, ws.bytes,
                               stream);
    }
    if (st != B200GPTQ_OK) Py_RETURN_NONE;   // the Python route repeats the call and reports the status
    return THPVariable_Wrap(std::move(y));
}

// Layer.run(x, module_dict).  No C++ exception leaves here: out of memory, or a tensor that has no address, is met again by
// the Python route, which raises it with its own type.
PyObject* layer_run(PyObject* self_, PyObject* const* args, Py_ssize_t nargs) {
    if (nargs != 2) { PyErr_SetString(PyExc_TypeError, "run(x, module_dict)"); return nullptr; }
    try {
        return run_prepared(reinterpret_cast<Layer*>(self_), args[0], args[1]);
    } catch (const std::exception&) {
        Py_RETURN_NONE;
    }
}

// Layer.set_gemv(rows, plan_owner, plan_handle, workspace_bytes)
PyObject* layer_set_gemv(PyObject* self_, PyObject* args) {
    Layer* self = reinterpret_cast<Layer*>(self_);
    int rows;
    PyObject* owner;
    unsigned long long handle, need;
    if (!PyArg_ParseTuple(args, "iOKK", &rows, &owner, &handle, &need)) return nullptr;
    if (rows < 1 || rows > kMaxGemvRows) { PyErr_SetString(PyExc_ValueError, "rows"); return nullptr; }
    GemvEntry& e = self->gemv[rows];
    Py_INCREF(owner);
    Py_XSETREF(e.owner, owner);
    e.plan = reinterpret_cast<const b200gptq_gemv_plan*>((uintptr_t)handle);
    e.need = (size_t)need;
    Py_RETURN_NONE;
}

// Layer(K, N, bits, group_size, device, module_dict, gemm_ok, gemv_rows, qweight_run, g_idx_run, x_perm)
PyObject* make_layer(PyTypeObject* type, PyObject* args) {
    int K, N, bits, group_size, device, gemm_ok, gemv_rows;
    PyObject *dict, *qw, *gi, *perm;
    if (!PyArg_ParseTuple(args, "iiiiiOpiOOO", &K, &N, &bits, &group_size, &device, &dict, &gemm_ok, &gemv_rows, &qw, &gi, &perm))
        return nullptr;
    PyObject* buffers = PyDict_Check(dict) ? PyDict_GetItem(dict, s_buffers) : nullptr;
    if (!buffers) { PyErr_SetString(PyExc_TypeError, "module_dict"); return nullptr; }
    PyObject *pq = PyDict_GetItem(buffers, s_qweight), *pg = PyDict_GetItem(buffers, s_g_idx),
             *pz = PyDict_GetItem(buffers, s_qzeros), *ps = PyDict_GetItem(buffers, s_scales);
    PyObject* bias = PyDict_GetItem(buffers, s_bias);
    if (!bias) bias = PyDict_GetItem(dict, s_bias);
    PyObject* tuning = PyDict_GetItem(dict, s_gemv_tuning);
    if (!pq || !pg || !pz || !ps || !THPVariable_Check(pq) || !THPVariable_Check(pg) || !THPVariable_Check(pz) || !THPVariable_Check(ps) ||
        (bias && bias != Py_None && !THPVariable_Check(bias))) {
        PyErr_SetString(PyExc_TypeError, "the module lacks a buffer");
        return nullptr;
    }
    // (the stored qweight and g_idx too: as long as they live nothing else can come to lie at their addresses)
    PyObject* keep = PyTuple_Pack(9, pq, pg, qw, gi, perm, pz, ps, bias ? bias : Py_None, tuning ? tuning : Py_None);
    if (!keep) return nullptr;
    Layer* self = reinterpret_cast<Layer*>(type->tp_alloc(type, 0));
    if (!self) { Py_DECREF(keep); return nullptr; }
    self->K = K; self->N = N; self->bits = bits; self->group_size = group_size; self->device = device;
    self->writes = writes_to(pq) + writes_to(pg) + writes_to(pz) + writes_to(ps);
    self->qweight_at = tensor_address(pq);
    self->g_idx_at = tensor_address(pg);
    self->qzeros = pz; self->scales = ps; self->bias = bias ? bias : Py_None; self->tuning = tuning;
    self->gemm_ok = gemm_ok != 0;
    self->gemv_rows = gemv_rows < kMaxGemvRows ? gemv_rows : kMaxGemvRows;
    self->qweight_run = static_cast<const int32_t*>(tensor_address(qw));
    self->g_idx_run = static_cast<const int32_t*>(tensor_address(gi));
    self->x_perm = static_cast<const int32_t*>(tensor_address(perm));
    self->qzeros_run = static_cast<const int32_t*>(tensor_address(pz));
    self->scales_run = tensor_address(ps);
    self->bias_run = tensor_address(bias);
    self->keep = keep;
    return reinterpret_cast<PyObject*>(self);
}

PyObject* layer_new(PyTypeObject* type, PyObject* args, PyObject*) {
    try {
        return make_layer(type, args);
    } catch (const std::exception& e) {      // a tensor without an address
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

void layer_dealloc(PyObject* self_) {
    Layer* self = reinterpret_cast<Layer*>(self_);
    for (auto& e : self->gemv) Py_XDECREF(e.owner);
    Py_XDECREF(self->keep);
    Py_TYPE(self_)->tp_free(self_);
}

PyMethodDef layer_methods[] = {
    {"run", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(layer_run)), METH_FASTCALL, nullptr},
    {"set_gemv", layer_set_gemv, METH_VARARGS, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyTypeObject LayerType = {PyVarObject_HEAD_INIT(nullptr, 0) "autogptq.tvm_b200._host.Layer", sizeof(Layer)};

// set_scratch(device, stream, tensor, bytes, in_graph)
PyObject* set_scratch(PyObject*, PyObject* args) {
    int device, in_graph;
    unsigned long long stream, bytes;
    PyObject* tensor;
    if (!PyArg_ParseTuple(args, "iKOKp", &device, &stream, &tensor, &bytes, &in_graph)) return nullptr;
    const void* address = nullptr;
    try {
        address = tensor_address(tensor);
    } catch (const std::exception&) {
    }
    if (!address) { PyErr_SetString(PyExc_TypeError, "set_scratch: a tensor"); return nullptr; }
    Scratch& s = (*g_scratch)[{device, (void*)(uintptr_t)stream}];
    PyObject* before = s.owner;
    Py_INCREF(tensor);
    s = Scratch{tensor, const_cast<void*>(address), (size_t)bytes, in_graph != 0};
    Py_XDECREF(before);
    Py_RETURN_NONE;
}
// scratch_use(device, stream): notes that the stream's scratch is handed out; (the stream is being captured, a graph may hold the
// address of the scratch)
PyObject* scratch_use(PyObject*, PyObject* args) {
    int device;
    unsigned long long stream;
    if (!PyArg_ParseTuple(args, "iK", &device, &stream)) return nullptr;
    bool capturing = false;
    try {
        capturing = is_capturing((cudaStream_t)(uintptr_t)stream);
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
    auto it = g_scratch->find({device, (void*)(uintptr_t)stream});
    if (it != g_scratch->end()) it->second.in_graph = it->second.in_graph || capturing;
    return Py_BuildValue("(NN)", PyBool_FromLong(capturing), PyBool_FromLong(it != g_scratch->end() && it->second.in_graph));
}
// zeros_outside_capture(device, bytes): zeroed memory that exists now, while a stream of this thread is being captured.  (An ordinary
// allocation would come from the graph's own memory, and be zeroed by the graph.)
PyObject* zeros_outside_capture(PyObject*, PyObject* args) {
    int device;
    long long bytes;
    if (!PyArg_ParseTuple(args, "iL", &device, &bytes)) return nullptr;
    try {
        const c10::cuda::CUDAGuard on((c10::DeviceIndex)device);
        const c10::cuda::CUDAStreamCaptureModeGuard relaxed{cudaStreamCaptureModeRelaxed};
        // (streams of the pool are handed out in turn: one of them may be the one that is captured)
        c10::cuda::CUDAStream side = c10::cuda::getStreamFromPool(false, (c10::DeviceIndex)device);
        for (int i = 0; i < 64 && is_capturing(side.stream()); ++i) side = c10::cuda::getStreamFromPool(false, (c10::DeviceIndex)device);
        const c10::cuda::CUDAStreamGuard beside(side);
        at::Tensor t = at::detail::empty_cuda({bytes}, at::kByte, at::Device(at::kCUDA, (c10::DeviceIndex)device), std::nullopt);
        C10_CUDA_CHECK(cudaMemsetAsync(t.mutable_data_ptr(), 0, (size_t)bytes, side.stream()));
        C10_CUDA_CHECK(cudaStreamSynchronize(side.stream()));
        return THPVariable_Wrap(std::move(t));
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}
// pack(weight, scales, zeros, g_idx, bits, copy_g_idx): QuantLinear.pack's (qweight, qzeros, scales, copy of g_idx or None) in one launch, or None
// where the Python route has more to do (another type, order, device or shape).
PyObject* pack_prepared(PyObject* const* args, Py_ssize_t nargs) {
    if (nargs != 6) { PyErr_SetString(PyExc_TypeError, "pack(weight, scales, zeros, g_idx, bits, copy_g_idx)"); return nullptr; }
    const at::Tensor* t[4];
    for (int i = 0; i < 4; ++i) {
        if (!THPVariable_Check(args[i])) Py_RETURN_NONE;
        t[i] = &THPVariable_Unpack(args[i]);
        if (t[i]->key_set().has_any(kNotPlain) || !t[i]->is_cuda() || !t[i]->is_contiguous()) Py_RETURN_NONE;
    }
    const at::Tensor &w = *t[0], &scales = *t[1], &zeros = *t[2], &g_idx = *t[3];
    const int bits = (int)PyLong_AsLong(args[4]), copy = PyObject_IsTrue(args[5]);
    if (PyErr_Occurred()) return nullptr;
    const auto type = w.scalar_type();
    const int dtype = type == at::kHalf ? B200GPTQ_F16 : (type == at::kBFloat16 ? B200GPTQ_BF16 : (type == at::kFloat ? B200GPTQ_F32 : -1));
    const int device = w.get_device();
    if (dtype < 0 || w.dim() != 2 || scales.dim() != 2 || scales.scalar_type() != at::kFloat || zeros.scalar_type() != at::kFloat ||
        g_idx.scalar_type() != at::kInt || g_idx.dim() != 1 || scales.get_device() != device || zeros.get_device() != device ||
        g_idx.get_device() != device || c10::cuda::current_device() != device)
        Py_RETURN_NONE;
    const int64_t N = w.size(0), K = w.size(1), G = scales.size(1);
    const void* wp = w.unsafeGetTensorImpl()->data();
    if (scales.size(0) != N || zeros.sizes() != scales.sizes() || g_idx.numel() != K || G < 1 || K < 32 || K % 32 || N < 32 || N % 32 ||
        K > INT32_MAX || N > INT32_MAX || ((uintptr_t)wp & 15u))
        Py_RETURN_NONE;
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
    const at::Device on(at::kCUDA, (c10::DeviceIndex)device);
    at::Tensor qweight, qzeros, scales16, g_copy;
    int st;
    {
        const WithoutGil released;
        qweight = at::detail::empty_cuda({K / 32 * bits, N}, at::kInt, on, std::nullopt);
        qzeros = at::detail::empty_cuda({G, N / 32 * bits}, at::kInt, on, std::nullopt);
        scales16 = at::detail::empty_cuda({G, N}, at::kHalf, on, std::nullopt);
        if (copy) g_copy = at::detail::empty_cuda({K}, at::kInt, on, std::nullopt);
        auto ints = [](at::Tensor& x) { return static_cast<int32_t*>(x.unsafeGetTensorImpl()->mutable_data()); };
        st = b200gptq_pack_linear_ex(wp, dtype, static_cast<const float*>(scales.unsafeGetTensorImpl()->data()),
                                     static_cast<const float*>(zeros.unsafeGetTensorImpl()->data()),
                                     static_cast<const int32_t*>(g_idx.unsafeGetTensorImpl()->data()), (int)K, (int)N, (int)G, bits,
                                     ints(qweight), ints(qzeros), scales16.unsafeGetTensorImpl()->mutable_data(),
                                     copy ? ints(g_copy) : nullptr, stream);
    }
    if (st != B200GPTQ_OK) Py_RETURN_NONE;   // the Python route repeats the call and reports the status
    PyObject* out[4] = {THPVariable_Wrap(std::move(qweight)), THPVariable_Wrap(std::move(qzeros)), THPVariable_Wrap(std::move(scales16)),
                        copy ? THPVariable_Wrap(std::move(g_copy)) : Py_NewRef(Py_None)};
    return Py_BuildValue("(NNNN)", out[0], out[1], out[2], out[3]);
}
PyObject* pack(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    try {
        return pack_prepared(args, nargs);
    } catch (const std::exception&) {        // out of memory: met again by the Python route, which raises it with its own type
        Py_RETURN_NONE;
    }
}
PyObject* set_scratch_source(PyObject*, PyObject* fn) {
    Py_INCREF(fn);
    Py_XSETREF(g_get_workspace, fn);
    Py_RETURN_NONE;
}

// ---- b200gptq_attn and b200gptq_adjust_logits: the checks that need tensors, the outputs' memory and the call.  There is no other route; what
//      is wrong is raised here, with the type that ops.py's other checks have. ----
struct Refusal { PyObject* type; std::string text; };
[[noreturn]] void refuse(PyObject* type, std::string text) { throw Refusal{type, std::move(text)}; }

const at::Tensor* tensor_or_none(PyObject* o, const char* name) {
    if (o == Py_None) return nullptr;
    if (!THPVariable_Check(o)) refuse(PyExc_TypeError, std::string(name) + " must be a tensor");
    const at::Tensor& t = THPVariable_Unpack(o);
    if (t.key_set().has_any(kNotPlain) || t.layout() != at::kStrided) refuse(PyExc_TypeError, std::string(name) + " must be a plain tensor");
    if (!t.is_cuda()) refuse(PyExc_RuntimeError, std::string(name) + " must be a CUDA tensor: the B200 GPTQ kernels have no CPU path");
    return &t;
}
const at::Tensor& tensor_of(PyObject* o, const char* name) {
    const at::Tensor* t = tensor_or_none(o, name);
    if (!t) refuse(PyExc_TypeError, std::string(name) + " must be a tensor");
    return *t;
}
void need(bool ok, const char* name, const char* what) {
    if (!ok) refuse(PyExc_ValueError, std::string(name) + " " + what);
}
void need_type(const at::Tensor& t, at::ScalarType type, const char* name) {
    if (t.scalar_type() != type) refuse(PyExc_TypeError, std::string(name) + " must be " + c10::toString(type) + ", got " + c10::toString(t.scalar_type()));
}
void need_device(const at::Tensor& t, int device, const char* name) {
    if (t.get_device() != device) refuse(PyExc_RuntimeError, std::string(name) + " is on another device");
}
// The arguments' names, in the order of the calls below.
constexpr int kArguments = 11;
constexpr const char* kWriteNames[] = {"k", "v", "cache.k", "cache.v", "cache.k_scales", "cache.v_scales", "pos", "counts", "cos", "sin", "q", "q_out", "k_out", "v_out"};
constexpr const char* kReadNames[] = {"cache.k", "cache.v", "cache.k_scales", "cache.v_scales", "lengths", "k_out", "v_out"};
constexpr const char* kAttnCacheNames[] = {"q", "cache.k", "cache.v", "cache.k_scales", "cache.v_scales", "pos", "window", "sinks", "counts", "scale", "out"};
constexpr const char* kSampleNames[] = {"logits", "uniform", "temperature", "top_k", "top_p", "min_p", "out"};
constexpr const char* kAttnNames[kArguments] = {"q", "k_prefix", "v_prefix", "k_cache", "v_cache", "pos", "window", "sinks", "counts", "scale", "out"};
constexpr const char* kLogitNames[kArguments] = {"logits", "history", "lengths", "prompt_lens", "repetition", "frequency", "presence", "bias_tokens", "bias_values", "mask", "out"};
// No argument asks for a derivative, backward or (a dual number, which knows no no_grad) forward: penalties and biases could as well as the logits.
void need_no_gradients(PyObject* const* args, const char* const* names, int count) {
    const bool backward = at::GradMode::is_enabled(), forward = c10::AutogradState::get_tls_state().get_fw_grad_mode();
    for (int i = 0; i < count; ++i) {
        // (THPVariable_Check asks Python about what is no tensor: 100 ns each)
        if (args[i] == Py_None || PyLong_CheckExact(args[i]) || PyFloat_CheckExact(args[i]) || !THPVariable_Check(args[i])) continue;
        const at::Tensor& t = THPVariable_Unpack(args[i]);
        if (backward && t.requires_grad()) refuse(PyExc_RuntimeError, std::string(names[i]) + " requires a gradient, and this operator has no backward pass");
        if (forward && t._fw_grad(0).defined()) refuse(PyExc_RuntimeError, std::string(names[i]) + " carries a tangent, and this operator has no forward-mode derivative");
    }
}
const void* data_of(const at::Tensor& t) { return t.unsafeGetTensorImpl()->data(); }
// The memory between a tensor's first and last element.
struct Memory {
    uintptr_t lo = 0, hi = 0;
    Memory() = default;
    explicit Memory(const at::Tensor& t) {
        int64_t last = 0;
        for (int64_t i = 0; i < t.dim(); ++i) {
            if (t.size(i) == 0) return;
            last += (t.size(i) - 1) * t.stride(i);
        }
        lo = (uintptr_t)data_of(t);
        hi = lo + (uintptr_t)((last + 1) * t.element_size());
    }
    bool meets(const Memory& o) const { return lo < o.hi && o.lo < hi; }
};
// Whether two tensors may have a byte in common.  Where one begins before the other ends they may still alternate (keys and values side by side in one allocation): seen modulo
// a stride of theirs, dimensions of which it divides the stride stay where they are, and what the others reach may lie apart.
bool alternate(const at::Tensor& x, const at::Tensor& y) {
    const uintptr_t at_x = (uintptr_t)data_of(x), at_y = (uintptr_t)data_of(y);
    auto reach = [](const at::Tensor& t, uintptr_t period) {
        const uintptr_t size = t.element_size();
        uintptr_t bytes = size;
        for (int64_t i = 0; i < t.dim(); ++i)
            if (t.size(i) > 1 && (uintptr_t)t.stride(i) * size % period) bytes += (uintptr_t)(t.size(i) - 1) * (uintptr_t)t.stride(i) * size;
        return bytes;
    };
    for (const at::Tensor* t : {&x, &y})
        for (int64_t i = 0; i < t->dim(); ++i) {
            const uintptr_t period = (uintptr_t)t->stride(i) * t->element_size();
            if (t->size(i) < 2 || period == 0) continue;
            const uintptr_t apart = at_y >= at_x ? (at_y - at_x) % period : (period - (at_x - at_y) % period) % period;        // from x on to y
            if (reach(x, period) <= apart && apart + reach(y, period) <= period) return true;
        }
    return false;
}
bool overlap(const at::Tensor& x, const at::Tensor& y) { return Memory(x).meets(Memory(y)) && !alternate(x, y); }
// Whether the elements of each dimension lie apart: a dimension's stride passes all that the dimensions of smaller strides reach.
bool apart_from_itself(const at::Tensor& t) {
    c10::SmallVector<std::pair<int64_t, int64_t>, 4> dims;         // (stride, size)
    for (int64_t i = 0; i < t.dim(); ++i)
        if (t.size(i) > 1) dims.emplace_back(t.stride(i), t.size(i));
    std::sort(dims.begin(), dims.end());
    int64_t reach = 1;
    for (auto [stride, size] : dims) {
        if (stride < reach) return false;
        reach += (size - 1) * stride;
    }
    return true;
}
int int_of(PyObject* o, const char* name) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) { PyErr_Clear(); refuse(PyExc_TypeError, std::string(name) + " must be an integer"); }
    need(v >= 0 && v <= (1 << 29), name, "is out of range");
    return (int)v;
}
// A tensor's strides by dimension; those of dimensions of size one are not used and count as 0.
template <size_t N> void strides_of(const at::Tensor& t, int64_t (&to)[N], const int (&dims)[N]) {
    for (size_t i = 0; i < N; ++i) to[i] = t.size(dims[i]) == 1 ? 0 : t.stride(dims[i]);
}
void need_rows(const at::Tensor& t, const char* name) {
    need(t.size(-1) == 1 || t.stride(-1) == 1, name, "must be dense in its last dimension");
    bool ok = ((uintptr_t)data_of(t) & 15u) == 0;
    for (int64_t i = 0; i + 1 < t.dim(); ++i) ok = ok && (t.size(i) == 1 || (t.stride(i) * (int64_t)t.element_size()) % 16 == 0);
    need(ok, name, "must have rows that begin at multiples of 16 bytes");
}
// int64 [batch]
const int64_t* whole_numbers(const at::Tensor* t, int device, int64_t batch, const char* name) {
    if (!t) return nullptr;
    need_type(*t, at::kLong, name);
    need_device(*t, device, name);
    need(t->dim() == 1 && t->size(0) == batch && (batch == 1 || t->stride(0) == 1), name, "must be int64, dense, one number for each sequence");
    return static_cast<const int64_t*>(data_of(*t));
}

// The output (one that was given counts a write in place), or a status code.
PyObject* answer(at::Tensor out, bool given, int st) {
    if (st != B200GPTQ_OK) return PyLong_FromLong(st);
    if (given && !out.is_inference()) out.unsafeGetTensorImpl()->bump_version();
    return THPVariable_Wrap(std::move(out));
}

// attn(q, k_prefix, v_prefix, k_cache, v_cache, pos, window, sinks, counts, scale, out): the output, or a status code
PyObject* attn_checked(PyObject* const* args) {
    const at::Tensor &q = tensor_of(args[0], "q"), &k = tensor_of(args[3], "k_cache"), &v = tensor_of(args[4], "v_cache"), &pos = tensor_of(args[5], "pos");
    const at::Tensor *kp = tensor_or_none(args[1], "k_prefix"), *vp = tensor_or_none(args[2], "v_prefix"), *counts = tensor_or_none(args[8], "counts"),
                     *given = tensor_or_none(args[10], "out");
    b200gptq_attn_args a = {};
    const int device = q.get_device();
    const at::ScalarType type = q.scalar_type();
    if (type != at::kHalf && type != at::kBFloat16) refuse(PyExc_TypeError, "q must be float16 or bfloat16");
    a.dtype = type == at::kHalf ? B200GPTQ_F16 : B200GPTQ_BF16;
    need(q.dim() == 4 && q.numel() > 0, "q", "must be [batch, tokens, heads, head_dim]");
    need(k.dim() == 4 && k.numel() > 0, "k_cache", "must be [batch, kv_heads, max_seq, head_dim]");
    const int64_t B = q.size(0), T = q.size(1), H = q.size(2), hd = q.size(3), KV = k.size(1), S = k.size(2);
    need(hd == 64 || hd == 128, "q", "must have heads of 64 or 128 dims");
    need(k.size(0) == B && k.size(3) == hd && H % KV == 0, "k_cache", "must be [batch, kv_heads, max_seq, head_dim], kv_heads a divisor of q's heads");
    need(v.sizes() == k.sizes(), "v_cache", "must have the shape of k_cache");
    need(B * T <= (1 << 29) && H <= (1 << 29) && B * T * (H / KV) <= (1 << 29) && S <= (1 << 29), "q", "is too large");
    for (auto [t, name] : {std::pair{&k, "k_cache"}, std::pair{&v, "v_cache"}}) {
        need_type(*t, type, name);
        need_device(*t, device, name);
        need_rows(*t, name);
    }
    need_rows(q, "q");
    need_type(pos, at::kLong, "pos");
    need_device(pos, device, "pos");
    need(pos.dim() == 1 && (pos.size(0) == B || pos.size(0) == 1) && (pos.size(0) == 1 || pos.stride(0) == 1), "pos", "must be int64, dense, one number or one for each sequence");
    a.pos = static_cast<const int64_t*>(data_of(pos));
    a.pos_each = pos.size(0) > 1;
    a.counts = whole_numbers(counts, device, B, "counts");
    a.batch = (int)B; a.tokens = (int)T; a.heads = (int)H; a.kv_heads = (int)KV; a.hd = (int)hd; a.max_seq = (int)S;
    a.q = data_of(q); a.k_cache = data_of(k); a.v_cache = data_of(v);
    strides_of(q, a.q_stride, {0, 1, 2});
    strides_of(k, a.k_stride, {0, 1, 2});
    strides_of(v, a.v_stride, {0, 1, 2});
    if (kp || vp) {
        need(kp && vp, "k_prefix", "and v_prefix come together");
        need(kp->dim() == 3 && kp->size(0) == KV && kp->size(2) == hd && kp->size(1) <= (1 << 29), "k_prefix", "must be [kv_heads, positions, head_dim]");
        need(vp->sizes() == kp->sizes(), "v_prefix", "must have the shape of k_prefix");
        for (auto [t, name] : {std::pair{kp, "k_prefix"}, std::pair{vp, "v_prefix"}}) {
            need_type(*t, type, name);
            need_device(*t, device, name);
        }
        a.prefix = (int)kp->size(1);
        if (a.prefix) {
            need_rows(*kp, "k_prefix");
            need_rows(*vp, "v_prefix");
            a.k_prefix = data_of(*kp); a.v_prefix = data_of(*vp);
            strides_of(*kp, a.k_prefix_stride, {0, 1});
            strides_of(*vp, a.v_prefix_stride, {0, 1});
        }
    } else {
        a.window = int_of(args[6], "window");
        a.sinks = int_of(args[7], "sinks");
        need(a.window >= 1, "window", "must be at least 1");
    }
    if (args[9] == Py_None) {
        a.scale = (float)(1.0 / std::sqrt((double)hd));
    } else {
        a.scale = (float)PyFloat_AsDouble(args[9]);
        if (PyErr_Occurred()) { PyErr_Clear(); refuse(PyExc_TypeError, "scale must be a number"); }
    }
    if (given) {
        need_type(*given, type, "out");
        need_device(*given, device, "out");
        need(given->sizes() == q.sizes(), "out", "must have the shape of q");
        need_rows(*given, "out");
        bool apart = !overlap(*given, q) && !overlap(*given, k) && !overlap(*given, v) && !overlap(*given, pos) && !(counts && overlap(*given, *counts));
        if (a.prefix) apart = apart && !overlap(*given, *kp) && !overlap(*given, *vp);
        need(apart && apart_from_itself(*given), "out", "must not overlap what is read, nor itself");
    }
    // (rows of padding that nobody has given a value)
    if (counts && !given) refuse(PyExc_ValueError, "counts needs out: the rows of padding keep what it holds");
    const at::Device on(at::kCUDA, (c10::DeviceIndex)device);
    const c10::cuda::OptionalCUDAGuard guard(c10::cuda::current_device() != device ? std::optional<at::Device>(on) : std::nullopt);
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
    Scratch ws;                 // (for its status word: what a wait that runs out raises)
    if (!scratch_for(device, stream, B200GPTQ_STATUS_BYTES, &ws)) return nullptr;
    const Held owner(ws.owner);
    a.status = reinterpret_cast<unsigned int*>(static_cast<char*>(ws.ptr) + B200GPTQ_STATUS_BYTES) - 1;
    at::Tensor out, scratch;
    int st;
    {
        const WithoutGil released;
        out = given ? *given : at::Tensor(at::detail::empty_cuda(q.sizes(), type, on, std::nullopt));
        a.out = out.unsafeGetTensorImpl()->mutable_data();
        strides_of(out, a.out_stride, {0, 1, 2});
        const int64_t bytes = b200gptq_attn_workspace_bytes(&a);
        if (bytes > 0) scratch = at::detail::empty_cuda({bytes}, at::kByte, on, std::nullopt);
        st = bytes < 0 ? (int)bytes : b200gptq_attn(&a, bytes > 0 ? scratch.unsafeGetTensorImpl()->mutable_data() : nullptr, (size_t)bytes, stream);
    }
    return answer(std::move(out), given != nullptr, st);
}

// adjust_logits(logits, history, lengths, prompt_lens, repetition, frequency, presence, bias_tokens, bias_values, mask, out)
PyObject* logits_checked(PyObject* const* args) {
    const at::Tensor& x = tensor_of(args[0], "logits");
    const char* const* names = kLogitNames;
    const at::Tensor* t[kArguments];
    const int device = x.get_device();
    for (int i = 1; i < kArguments; ++i) {
        t[i] = tensor_or_none(args[i], names[i]);
        if (t[i]) need_device(*t[i], device, names[i]);
    }
    b200gptq_logit_args a = {};
    const at::ScalarType type = x.scalar_type();
    if (type != at::kHalf && type != at::kBFloat16 && type != at::kFloat) refuse(PyExc_TypeError, "logits must be float16, bfloat16 or float32");
    a.dtype = type == at::kHalf ? B200GPTQ_F16 : type == at::kBFloat16 ? B200GPTQ_BF16 : B200GPTQ_F32;
    need(x.dim() == 2 && x.numel() > 0 && (x.size(1) == 1 || x.stride(1) == 1) && x.size(0) <= INT32_MAX && x.size(1) <= (1 << 30), "logits", "must be [rows, vocab], dense in its last dimension");
    const int64_t R = x.size(0), V = x.size(1);
    a.rows = (int)R; a.vocab = (int)V;
    a.logits = data_of(x);
    a.logits_stride = R == 1 ? 0 : x.stride(0);
    need((t[1] != nullptr) == (t[2] != nullptr), "history", "and lengths come together");
    need(t[1] || (!t[3] && !t[4] && !t[5] && !t[6]), "history", "is needed for penalties");
    if (t[1]) {
        need_type(*t[1], at::kLong, "history");
        need(t[1]->dim() == 2 && t[1]->size(0) == R && t[1]->size(1) < (1 << 30) && (t[1]->size(1) <= 1 || t[1]->stride(1) == 1), "history", "must be [rows, positions], dense in its last dimension");
        a.history_len = (int)t[1]->size(1);
        a.history = a.history_len ? static_cast<const int64_t*>(data_of(*t[1])) : nullptr;
        a.history_stride = R == 1 ? 0 : t[1]->stride(0);
    }
    a.lengths = whole_numbers(t[2], device, R, "lengths");
    a.prompt_lens = whole_numbers(t[3], device, R, "prompt_lens");
    const float** params[3] = {&a.repetition, &a.frequency, &a.presence};
    for (int i = 4; i < 7; ++i)
        if (t[i]) {
            need_type(*t[i], at::kFloat, names[i]);
            need(t[i]->dim() == 1 && t[i]->size(0) == R && (R == 1 || t[i]->stride(0) == 1), names[i], "must be float32, dense, one number for each row");
            *params[i - 4] = static_cast<const float*>(data_of(*t[i]));
        }
    need((t[7] != nullptr) == (t[8] != nullptr), "bias_tokens", "and bias_values come together");
    if (t[7]) {
        need_type(*t[7], at::kLong, "bias_tokens");
        need_type(*t[8], at::kFloat, "bias_values");
        need(t[7]->dim() == 2 && t[7]->size(0) == R && t[7]->size(1) < (1 << 30) && t[7]->is_contiguous(), "bias_tokens", "must be [rows, entries], contiguous");
        need(t[8]->sizes() == t[7]->sizes() && t[8]->is_contiguous(), "bias_values", "must have the shape of bias_tokens, contiguous");
        a.biases = (int)t[7]->size(1);
        if (a.biases) { a.bias_tokens = static_cast<const int64_t*>(data_of(*t[7])); a.bias_values = static_cast<const float*>(data_of(*t[8])); }
    }
    if (t[9]) {
        need_type(*t[9], at::kInt, "mask");
        need(t[9]->dim() == 2 && (t[9]->size(0) == R || t[9]->size(0) == 1) && t[9]->size(1) == (V + 31) / 32 && (t[9]->size(1) == 1 || t[9]->stride(1) == 1), "mask",
             "must be [rows or 1, ceil(vocab / 32)], dense in its last dimension");
        a.mask = static_cast<const int32_t*>(data_of(*t[9]));
        a.mask_stride = t[9]->size(0) == 1 ? 0 : t[9]->stride(0);
    }
    if (t[10]) {
        const at::Tensor& o = *t[10];
        need_type(o, type, "out");
        need(o.sizes() == x.sizes() && (V == 1 || o.stride(1) == 1) && (R == 1 || o.stride(0) >= V), "out", "must have the shape of logits, rows apart and dense in its last dimension");
        bool apart = (data_of(o) == data_of(x) && (R == 1 || o.stride(0) == x.stride(0))) || !overlap(o, x);
        for (int i = 1; i < 10; ++i) apart = apart && !(t[i] && overlap(o, *t[i]));
        need(apart, "out", "must be logits itself or overlap nothing that is read");
    }
    const at::Device on(at::kCUDA, (c10::DeviceIndex)device);
    const c10::cuda::OptionalCUDAGuard guard(c10::cuda::current_device() != device ? std::optional<at::Device>(on) : std::nullopt);
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
    at::Tensor out;
    int st;
    {
        const WithoutGil released;
        out = t[10] ? *t[10] : at::Tensor(at::detail::empty_cuda({R, V}, type, on, std::nullopt));
        a.out = out.unsafeGetTensorImpl()->mutable_data();
        a.out_stride = R == 1 ? 0 : out.stride(0);
        st = b200gptq_adjust_logits(&a, stream);
    }
    return answer(std::move(out), t[10] != nullptr, st);
}

// ---- the cache held in 4 bits ----
// Fills `c` from the tensors of an ops.QuantCache: codes, codes, constants, constants.  `written`: its elements have to lie apart.
void cache_of(const at::Tensor* const (&t)[4], const char* const* names, bool written, b200gptq_cache4& c) {
    const at::Tensor &k = *t[0], &scales = *t[2];
    const int device = k.get_device();
    const at::ScalarType type = scales.scalar_type();
    if (type != at::kHalf && type != at::kBFloat16) refuse(PyExc_TypeError, std::string(names[2]) + " must be float16 or bfloat16");
    need(k.dim() == 4 && k.numel() > 0, names[0], "must be [batch, kv_heads, max_seq, head_dim / 2]");
    const int64_t B = k.size(0), KV = k.size(1), S = k.size(2), hd = 2 * k.size(3);
    need(hd == 64 || hd == 128, names[0], "must have heads of 64 or 128 dims");
    need(B <= (1 << 29) && KV <= (1 << 29) && S <= (1 << 29), names[0], "is too large");
    need(scales.dim() == 5 && scales.size(0) == B && scales.size(1) == KV && scales.size(2) == S && scales.size(4) == 2 &&
             (scales.size(3) * 32 == hd || scales.size(3) * 64 == hd), names[2], "must be [batch, kv_heads, max_seq, head_dim / group, 2] with groups of 32 or 64");
    need(t[1]->sizes() == k.sizes(), names[1], "must have the shape of the keys' codes");
    need(t[3]->sizes() == scales.sizes(), names[3], "must have the shape of the keys' constants");
    const int64_t groups = scales.size(3);
    void** at[4] = {&c.k, &c.v, &c.k_scales, &c.v_scales};
    int64_t(*stride[4])[3] = {&c.k_stride, &c.v_stride, &c.k_scale_stride, &c.v_scale_stride};
    for (int i = 0; i < 4; ++i) {
        const at::Tensor& x = *t[i];
        need_type(x, i < 2 ? at::kByte : type, names[i]);
        need_device(x, device, names[i]);
        if (i < 2) {
            need_rows(x, names[i]);
        } else {
            bool ok = x.stride(4) == 1 && (groups == 1 || x.stride(3) == 2) && ((uintptr_t)data_of(x) & (uintptr_t)(4 * groups - 1)) == 0;
            for (int d = 0; d < 3; ++d) ok = ok && (x.size(d) == 1 || x.stride(d) % (2 * groups) == 0);
            need(ok, names[i], "must be dense in its last two dimensions, with rows that begin at multiples of their own size");
        }
        need(!written || apart_from_itself(x), names[i], "must not overlap itself");
        *at[i] = const_cast<void*>(data_of(x));
        strides_of(x, *stride[i], {0, 1, 2});
    }
    c.dtype = type == at::kHalf ? B200GPTQ_F16 : B200GPTQ_BF16;
    c.batch = (int)B; c.kv_heads = (int)KV; c.max_seq = (int)S; c.hd = (int)hd; c.group = (int)(hd / groups);
}
void positions_of(const at::Tensor& pos, int device, int64_t batch, const int64_t** at, int* each) {
    need_type(pos, at::kLong, "pos");
    need_device(pos, device, "pos");
    need(pos.dim() == 1 && (pos.size(0) == batch || pos.size(0) == 1) && (pos.size(0) == 1 || pos.stride(0) == 1), "pos", "must be int64, dense, one number or one for each sequence");
    *at = static_cast<const int64_t*>(data_of(pos));
    *each = pos.size(0) > 1;
}
void wrote(const at::Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// cache_write(k, v, cache.k, cache.v, cache.k_scales, cache.v_scales, pos, counts, cos, sin, q, q_out, k_out, v_out): q_out or None, or a status code
PyObject* write_checked(PyObject* const* args) {
    const at::Tensor* t[14];
    for (int i = 0; i < 14; ++i) t[i] = i < 7 ? &tensor_of(args[i], kWriteNames[i]) : tensor_or_none(args[i], kWriteNames[i]);
    const char* const* names = kWriteNames;
    b200gptq_cache_write_args a = {};
    const at::Tensor* const cache[4] = {t[2], t[3], t[4], t[5]};
    cache_of(cache, names + 2, true, a.cache);
    const int device = t[2]->get_device();
    const at::ScalarType type = t[4]->scalar_type();
    const int64_t B = a.cache.batch, KV = a.cache.kv_heads, hd = a.cache.hd;
    need(t[0]->dim() == 4 && t[0]->numel() > 0 && t[0]->size(0) == B && t[0]->size(2) == KV && t[0]->size(3) == hd, "k", "must be [batch, tokens, kv_heads, head_dim] of the cache's sizes");
    const int64_t T = t[0]->size(1);
    need(T <= (1 << 29), "k", "is too large");
    need((t[8] != nullptr) == (t[9] != nullptr), "cos", "and sin come together");
    need((t[10] != nullptr) == (t[11] != nullptr), "q", "and q_out come together");
    need((t[12] != nullptr) == (t[13] != nullptr), "k_out", "and v_out come together");
    need(!t[10] || t[8], "q", "is there to be rotated: cos and sin are missing");
    positions_of(*t[6], device, B, &a.pos, &a.pos_each);
    a.counts = whole_numbers(t[7], device, B, "counts");
    if (t[8]) {
        for (int i : {8, 9}) {
            need_type(*t[i], type, names[i]);
            need_device(*t[i], device, names[i]);
            need(t[i]->dim() == 2 && t[i]->numel() > 0 && t[i]->size(1) * 2 == hd && t[i]->size(0) <= (1 << 29) && t[i]->is_contiguous() && ((uintptr_t)data_of(*t[i]) & 15u) == 0, names[i],
                 "must be [positions, head_dim / 2], contiguous and on 16 bytes");
        }
        need(t[9]->size(0) == t[8]->size(0), "sin", "must have the shape of cos");
        a.cos_t = data_of(*t[8]); a.sin_t = data_of(*t[9]);
        a.angles = (int)t[8]->size(0);
    }
    if (t[10]) {
        need(t[10]->dim() == 4 && t[10]->numel() > 0 && t[10]->size(0) == B && t[10]->size(1) == T && t[10]->size(3) == hd && t[10]->size(2) <= (1 << 29), "q", "must be [batch, tokens, heads, head_dim]");
        need(t[11]->sizes() == t[10]->sizes(), "q_out", "must have the shape of q");
        a.heads = (int)t[10]->size(2);
    }
    struct { int i; const void** at; int64_t (*stride)[3]; } rows[6] = {{0, &a.k, &a.k_stride}, {1, &a.v, &a.v_stride}, {10, &a.q, &a.q_stride},
        {11, const_cast<const void**>(&a.q_out), &a.q_out_stride}, {12, const_cast<const void**>(&a.k_out), &a.k_out_stride}, {13, const_cast<const void**>(&a.v_out), &a.v_out_stride}};
    for (auto& r : rows) {
        const at::Tensor* x = t[r.i];
        if (!x) continue;
        need(r.i == 10 || r.i == 11 || x->sizes() == t[0]->sizes(), names[r.i], "must have the shape of k");
        need_type(*x, type, names[r.i]);
        need_device(*x, device, names[r.i]);
        need_rows(*x, names[r.i]);
        *r.at = data_of(*x);
        strides_of(*x, *r.stride, {0, 1, 2});
    }
    // what is written overlaps nothing else: the cache (2 .. 5, whose parts have been found apart from themselves), q_out, k_out, v_out
    Memory memory[14];
    for (int i = 0; i < 14; ++i)
        if (t[i]) memory[i] = Memory(*t[i]);
    for (int i : {2, 3, 4, 5, 11, 12, 13}) {
        if (!t[i]) continue;
        bool apart = i < 6 || apart_from_itself(*t[i]);
        for (int j = 0; j < 14; ++j) apart = apart && (j == i || !memory[i].meets(memory[j]) || alternate(*t[i], *t[j]));
        need(apart, names[i], "must not overlap another tensor, nor itself");
    }
    a.tokens = (int)T;
    const at::Device on(at::kCUDA, (c10::DeviceIndex)device);
    const c10::cuda::OptionalCUDAGuard guard(c10::cuda::current_device() != device ? std::optional<at::Device>(on) : std::nullopt);
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
    int st;
    {
        const WithoutGil released;
        st = b200gptq_cache_write(&a, stream);
    }
    if (st != B200GPTQ_OK) return PyLong_FromLong(st);
    for (int i : {2, 3, 4, 5, 11, 12, 13})
        if (t[i]) wrote(*t[i]);
    if (!t[11]) Py_RETURN_NONE;
    Py_INCREF(args[11]);
    return args[11];
}

// cache_read(cache.k, cache.v, cache.k_scales, cache.v_scales, lengths, k_out, v_out): (k, v), or a status code
PyObject* read_checked(PyObject* const* args) {
    const at::Tensor* t[7];
    for (int i = 0; i < 7; ++i) t[i] = i < 4 ? &tensor_of(args[i], kReadNames[i]) : tensor_or_none(args[i], kReadNames[i]);
    b200gptq_cache_read_args a = {};
    const at::Tensor* const cache[4] = {t[0], t[1], t[2], t[3]};
    cache_of(cache, kReadNames, false, a.cache);
    const int device = t[0]->get_device();
    const at::ScalarType type = t[2]->scalar_type();
    const int64_t shape[4] = {a.cache.batch, a.cache.kv_heads, a.cache.max_seq, a.cache.hd};
    a.lengths = whole_numbers(t[4], device, a.cache.batch, "lengths");
    need((t[5] != nullptr) == (t[6] != nullptr), "k_out", "and v_out come together");
    if (t[4] && !t[5]) refuse(PyExc_ValueError, "lengths needs k_out and v_out: the rows behind them keep what they hold");
    for (int i : {5, 6}) {
        if (!t[i]) continue;
        need_type(*t[i], type, kReadNames[i]);
        need_device(*t[i], device, kReadNames[i]);
        need(t[i]->sizes() == at::IntArrayRef(shape), kReadNames[i], "must be [batch, kv_heads, max_seq, head_dim] of the cache's sizes");
        need_rows(*t[i], kReadNames[i]);
        bool apart = apart_from_itself(*t[i]);
        for (int j = 0; j < 7; ++j) apart = apart && (j == i || !t[j] || !overlap(*t[i], *t[j]));
        need(apart, kReadNames[i], "must not overlap another tensor, nor itself");
    }
    const at::Device on(at::kCUDA, (c10::DeviceIndex)device);
    const c10::cuda::OptionalCUDAGuard guard(c10::cuda::current_device() != device ? std::optional<at::Device>(on) : std::nullopt);
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
    at::Tensor out[2];
    int st;
    {
        const WithoutGil released;
        for (int i = 0; i < 2; ++i) out[i] = t[5 + i] ? *t[5 + i] : at::Tensor(at::detail::empty_cuda(at::IntArrayRef(shape), type, on, std::nullopt));
        a.k_out = out[0].unsafeGetTensorImpl()->mutable_data();
        a.v_out = out[1].unsafeGetTensorImpl()->mutable_data();
        strides_of(out[0], a.k_out_stride, {0, 1, 2});
        strides_of(out[1], a.v_out_stride, {0, 1, 2});
        st = b200gptq_cache_read(&a, stream);
    }
    if (st != B200GPTQ_OK) return PyLong_FromLong(st);
    PyObject* pair = PyTuple_New(2);
    for (int i = 0; pair && i < 2; ++i) {
        if (t[5 + i]) wrote(out[i]);
        PyTuple_SET_ITEM(pair, i, THPVariable_Wrap(std::move(out[i])));
    }
    return pair;
}

// attn_cache(q, cache.k, cache.v, cache.k_scales, cache.v_scales, pos, window, sinks, counts, scale, out): the output, or a status code
PyObject* attn_cache_checked(PyObject* const* args) {
    const at::Tensor &q = tensor_of(args[0], "q"), &pos = tensor_of(args[5], "pos");
    const at::Tensor* cache[4];
    for (int i = 0; i < 4; ++i) cache[i] = &tensor_of(args[1 + i], kAttnCacheNames[1 + i]);
    const at::Tensor *counts = tensor_or_none(args[8], "counts"), *given = tensor_or_none(args[10], "out");
    b200gptq_attn_cache_args a = {};
    cache_of(cache, kAttnCacheNames + 1, false, a.cache);
    const int device = cache[0]->get_device();
    const at::ScalarType type = cache[2]->scalar_type();
    const int64_t B = a.cache.batch, KV = a.cache.kv_heads;
    need_type(q, type, "q");
    need_device(q, device, "q");
    need(q.dim() == 4 && q.numel() > 0 && q.size(0) == B && q.size(3) == a.cache.hd && q.size(2) % KV == 0, "q", "must be [batch, tokens, heads, head_dim] of the cache's sizes, heads a multiple of its heads");
    const int64_t T = q.size(1), H = q.size(2);
    need(B * T <= (1 << 29) && H <= (1 << 29) && B * T * (H / KV) <= (1 << 29), "q", "is too large");
    need_rows(q, "q");
    positions_of(pos, device, B, &a.pos, &a.pos_each);
    a.counts = whole_numbers(counts, device, B, "counts");
    a.tokens = (int)T; a.heads = (int)H;
    a.q = data_of(q);
    strides_of(q, a.q_stride, {0, 1, 2});
    a.sinks = int_of(args[7], "sinks");
    if (args[6] != Py_None) {
        a.window = int_of(args[6], "window");
        need(a.window >= 1, "window", "must be at least 1");
    }
    need(a.window || !a.sinks, "sinks", "go with a window");
    if (args[9] == Py_None) {
        a.scale = (float)(1.0 / std::sqrt((double)a.cache.hd));
    } else {
        a.scale = (float)PyFloat_AsDouble(args[9]);
        if (PyErr_Occurred()) { PyErr_Clear(); refuse(PyExc_TypeError, "scale must be a number"); }
    }
    if (given) {
        need_type(*given, type, "out");
        need_device(*given, device, "out");
        need(given->sizes() == q.sizes(), "out", "must have the shape of q");
        need_rows(*given, "out");
        bool apart = !overlap(*given, q) && !overlap(*given, pos) && !(counts && overlap(*given, *counts));
        for (const at::Tensor* t : cache) apart = apart && !overlap(*given, *t);
        need(apart && apart_from_itself(*given), "out", "must not overlap what is read, nor itself");
    }
    if (counts && !given) refuse(PyExc_ValueError, "counts needs out: the rows of padding keep what it holds");
    const at::Device on(at::kCUDA, (c10::DeviceIndex)device);
    const c10::cuda::OptionalCUDAGuard guard(c10::cuda::current_device() != device ? std::optional<at::Device>(on) : std::nullopt);
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
    Scratch ws;                 // (for its status word: what a wait that runs out raises)
    if (!scratch_for(device, stream, B200GPTQ_STATUS_BYTES, &ws)) return nullptr;
    const Held owner(ws.owner);
    a.status = reinterpret_cast<unsigned int*>(static_cast<char*>(ws.ptr) + B200GPTQ_STATUS_BYTES) - 1;
    at::Tensor out, scratch;
    int st;
    {
        const WithoutGil released;
        out = given ? *given : at::Tensor(at::detail::empty_cuda(q.sizes(), type, on, std::nullopt));
        a.out = out.unsafeGetTensorImpl()->mutable_data();
        strides_of(out, a.out_stride, {0, 1, 2});
        const int64_t bytes = b200gptq_attn_cache_workspace_bytes(&a);
        if (bytes > 0) scratch = at::detail::empty_cuda({bytes}, at::kByte, on, std::nullopt);
        st = bytes < 0 ? (int)bytes : b200gptq_attn_cache(&a, bytes > 0 ? scratch.unsafeGetTensorImpl()->mutable_data() : nullptr, (size_t)bytes, stream);
    }
    return answer(std::move(out), given != nullptr, st);
}

// sample(logits, uniform, temperature, top_k, top_p, min_p, out): the tokens, or a status code
PyObject* sample_checked(PyObject* const* args) {
    const at::Tensor& x = tensor_of(args[0], "logits");
    const at::Tensor* t[7] = {&x, &tensor_of(args[1], "uniform")};
    const int device = x.get_device();
    for (int i = 1; i < 7; ++i) {
        if (i > 1) t[i] = tensor_or_none(args[i], kSampleNames[i]);
        if (t[i]) need_device(*t[i], device, kSampleNames[i]);
    }
    b200gptq_sample_args a = {};
    const at::ScalarType type = x.scalar_type();
    if (type != at::kHalf && type != at::kBFloat16 && type != at::kFloat) refuse(PyExc_TypeError, "logits must be float16, bfloat16 or float32");
    a.dtype = type == at::kHalf ? B200GPTQ_F16 : type == at::kBFloat16 ? B200GPTQ_BF16 : B200GPTQ_F32;
    need(x.dim() == 2 && x.numel() > 0 && (x.size(1) == 1 || x.stride(1) == 1), "logits", "must be [rows, vocab], dense in its last dimension");
    need(x.size(1) <= (1 << 18) && x.size(0) <= (1 << 27), "logits", "is too large: 2^18 tokens at most");
    const int64_t R = x.size(0);
    a.rows = (int)R; a.vocab = (int)x.size(1);
    a.logits = data_of(x);
    a.logits_stride = R == 1 ? 0 : x.stride(0);
    const float** numbers[7] = {nullptr, &a.uniform, &a.temperature, nullptr, &a.top_p, &a.min_p, nullptr};
    for (int i : {1, 2, 4, 5})
        if (t[i]) {
            need_type(*t[i], at::kFloat, kSampleNames[i]);
            need(t[i]->dim() == 1 && t[i]->size(0) == R && (R == 1 || t[i]->stride(0) == 1), kSampleNames[i], "must be float32, dense, one number for each row");
            *numbers[i] = static_cast<const float*>(data_of(*t[i]));
        }
    for (int i : {3, 6})
        if (t[i]) {
            need_type(*t[i], at::kLong, kSampleNames[i]);
            need(t[i]->dim() == 1 && t[i]->size(0) == R && (R == 1 || t[i]->stride(0) == 1), kSampleNames[i], "must be int64, dense, one number for each row");
        }
    if (t[3]) a.top_k = static_cast<const int64_t*>(data_of(*t[3]));
    for (int i = 0; i < 6 && t[6]; ++i) need(!t[i] || !overlap(*t[6], *t[i]), "out", "must overlap nothing that is read");
    const at::Device on(at::kCUDA, (c10::DeviceIndex)device);
    const c10::cuda::OptionalCUDAGuard guard(c10::cuda::current_device() != device ? std::optional<at::Device>(on) : std::nullopt);
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
    at::Tensor out;
    int st;
    {
        const WithoutGil released;
        out = t[6] ? *t[6] : at::Tensor(at::detail::empty_cuda({R}, at::kLong, on, std::nullopt));
        a.out = static_cast<int64_t*>(out.unsafeGetTensorImpl()->mutable_data());
        st = b200gptq_sample(&a, stream);
    }
    return answer(std::move(out), t[6] != nullptr, st);
}

template <int N>
PyObject* raising(PyObject* (*call)(PyObject* const*), const char* const (&names)[N], PyObject* const* args, Py_ssize_t nargs) {
    if (nargs != N) { PyErr_SetString(PyExc_TypeError, (std::to_string(N) + " arguments").c_str()); return nullptr; }
    try {
        need_no_gradients(args, names, N);
        return call(args);
    } catch (const Refusal& r) {
        PyErr_SetString(r.type, r.text.c_str());
    } catch (const c10::OutOfMemoryError& e) {
        const Held torch(PyImport_ImportModule("torch"), true), type(torch.o ? PyObject_GetAttrString(torch.o, "OutOfMemoryError") : nullptr, true);
        if (type.o) PyErr_SetString(type.o, e.what_without_backtrace());
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}
PyObject* attn(PyObject*, PyObject* const* args, Py_ssize_t nargs) { return raising(attn_checked, kAttnNames, args, nargs); }
PyObject* adjust_logits(PyObject*, PyObject* const* args, Py_ssize_t nargs) { return raising(logits_checked, kLogitNames, args, nargs); }
PyObject* cache_write(PyObject*, PyObject* const* args, Py_ssize_t nargs) { return raising(write_checked, kWriteNames, args, nargs); }
PyObject* attn_cache(PyObject*, PyObject* const* args, Py_ssize_t nargs) { return raising(attn_cache_checked, kAttnCacheNames, args, nargs); }
PyObject* sample(PyObject*, PyObject* const* args, Py_ssize_t nargs) { return raising(sample_checked, kSampleNames, args, nargs); }
PyObject* cache_read(PyObject*, PyObject* const* args, Py_ssize_t nargs) { return raising(read_checked, kReadNames, args, nargs); }

PyMethodDef module_methods[] = {
    {"attn", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(attn)), METH_FASTCALL, nullptr},
    {"adjust_logits", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(adjust_logits)), METH_FASTCALL, nullptr},
    {"cache_write", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(cache_write)), METH_FASTCALL, nullptr},
    {"attn_cache", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(attn_cache)), METH_FASTCALL, nullptr},
    {"sample", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(sample)), METH_FASTCALL, nullptr},
    {"cache_read", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(cache_read)), METH_FASTCALL, nullptr},
    {"pack", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(pack)), METH_FASTCALL, nullptr},
    {"set_scratch", set_scratch, METH_VARARGS, nullptr},
    {"set_scratch_source", set_scratch_source, METH_O, nullptr},
    {"scratch_use", scratch_use, METH_VARARGS, nullptr},
    {"zeros_outside_capture", zeros_outside_capture, METH_VARARGS, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, module_methods};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) {
    g_scratch = new std::unordered_map<std::pair<int, void*>, Scratch, KeyHash>();
    s_buffers = PyUnicode_InternFromString("_buffers");
    s_qweight = PyUnicode_InternFromString("qweight");
    s_g_idx = PyUnicode_InternFromString("g_idx");
    s_qzeros = PyUnicode_InternFromString("qzeros");
    s_scales = PyUnicode_InternFromString("scales");
    s_bias = PyUnicode_InternFromString("bias");
    s_gemv_tuning = PyUnicode_InternFromString("gemv_tuning");
    LayerType.tp_flags = Py_TPFLAGS_DEFAULT;
    LayerType.tp_new = layer_new;
    LayerType.tp_dealloc = layer_dealloc;
    LayerType.tp_methods = layer_methods;
    if (PyType_Ready(&LayerType) < 0) return nullptr;
    PyObject* m = PyModule_Create(&module_def);
    if (!m) return nullptr;
    Py_INCREF(&LayerType);
    if (PyModule_AddObject(m, "Layer", reinterpret_cast<PyObject*>(&LayerType)) < 0) return nullptr;
    return m;
}
