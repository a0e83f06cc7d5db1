// hawk_bind.cpp — a stage's call from Python: the call's planes checked against
// the plan of the call before, their addresses put into the job, the entry
// called, in one crossing.
//
// A call's tensors mostly have the names, types, shapes and strides of the last
// ones.  Asked for one by one from Python those cost 0.35 us a plane: a recurrence's
// step of 64 x 2048 bfloat16 channels took 7.8 us a call (4.9 so) and the policy loss
// of 200 rows of 48 logits, with its planes, 9.8 (6.3).

#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <cstring>
#include <map>
#include <mutex>
#include <utility>
#include <vector>

namespace {

constexpr size_t kMostWords = 64;
typedef int (*Entry)(const void* job, void* scratch, void* stream);
typedef int (*PlainEntry)(const void* job, void* stream);
typedef int (*Capturing)(void* stream);

struct Plane {
    PyObject* name;          // held; a call's names are the same objects
    bool value;              // an int, put into the job as it is
    at::ScalarType type;
    std::vector<int64_t> sizes, strides;
    int64_t word;            // -1: checked, not bound
};

struct Space {
    uint64_t stream, scratch, state;
    std::mutex* launches;
};

struct Plan {
    void* entry;
    bool plain;              // the entry takes no scratch
    bool needs_space;
    int device;
    Capturing capturing;     // or NULL: no call is captured
    int64_t state_word;
    std::vector<uint64_t> job;
    std::vector<Plane> planes;
    std::vector<std::pair<int, int>> apart;
    std::vector<Space> spaces;
};

struct Call {
    PyObject_HEAD
    Plan* plan;
};

// Calls on one stream share its scratch, so each one's launches stay together; a
// launch that blocks holds no other stream's.  (Found under the interpreter's lock.)
std::mutex* launches_of(int device, uint64_t stream) {
    static auto& all = *new std::map<std::pair<int, uint64_t>, std::mutex>;      // outlives every thread
    return &all[{device, stream}];
}

int enter(const Plan& plan, const uint64_t* job, uint64_t scratch, uint64_t stream, std::mutex* launches) {
    int rc;
    Py_BEGIN_ALLOW_THREADS
    {
        std::unique_lock<std::mutex> hold;
        if (launches) hold = std::unique_lock<std::mutex>(*launches);
        void* s = reinterpret_cast<void*>(stream);
        rc = plan.plain ? reinterpret_cast<PlainEntry>(plan.entry)(job, s)
                        : reinterpret_cast<Entry>(plan.entry)(job, reinterpret_cast<void*>(scratch), s);
    }
    Py_END_ALLOW_THREADS
    return rc;
}

// Call(entry, plain, needs_space, device, job, state_word, planes, apart, capturing):
// planes is a tuple of (name, tensor or None, word), apart one of (plane, plane)
// positions, capturing (may be left out) tells whether a stream is under capture.
int call_init(PyObject* self, PyObject* args, PyObject*) {
    unsigned long long entry, capturing = 0;
    int plain, needs_space, device;
    const char* job;
    Py_ssize_t job_bytes;
    long long state_word;
    PyObject *planes, *apart;
    if (!PyArg_ParseTuple(args, "Kppiy#LO!O!|K", &entry, &plain, &needs_space, &device, &job, &job_bytes, &state_word,
                          &PyTuple_Type, &planes, &PyTuple_Type, &apart, &capturing))
        return -1;
    if (job_bytes % 8 != 0 || static_cast<size_t>(job_bytes) / 8 > kMostWords) {
        PyErr_SetString(PyExc_ValueError, "a job of whole words, 64 at most");
        return -1;
    }
    Plan* plan = new Plan;
    reinterpret_cast<Call*>(self)->plan = plan;
    plan->entry = reinterpret_cast<void*>(entry);
    plan->plain = plain;
    plan->needs_space = needs_space;
    plan->device = device;
    plan->capturing = reinterpret_cast<Capturing>(capturing);
    plan->state_word = state_word;
    plan->job.resize(job_bytes / 8);
    std::memcpy(plan->job.data(), job, job_bytes);
    const int64_t words = job_bytes / 8;
    bool fits = state_word < words;
    try {
        for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(planes); ++i) {
            PyObject *name, *x;
            long long word;
            if (!PyArg_ParseTuple(PyTuple_GET_ITEM(planes, i), "UOL", &name, &x, &word)) return -1;
            Plane p{name, x == Py_None, at::ScalarType::Undefined, {}, {}, word};
            if (!p.value) {
                if (!THPVariable_Check(x)) {
                    PyErr_SetString(PyExc_TypeError, "a plane is a tensor");
                    return -1;
                }
                const at::Tensor& t = THPVariable_Unpack(x);
                p.type = t.scalar_type();
                p.sizes = t.sizes().vec();
                p.strides = t.strides().vec();
            }
            fits = fits && word < words;
            Py_INCREF(name);
            plan->planes.push_back(std::move(p));
        }
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_TypeError, e.what());
        return -1;
    }
    const Py_ssize_t count = PyTuple_GET_SIZE(planes);
    for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(apart); ++i) {
        int one, two;
        if (!PyArg_ParseTuple(PyTuple_GET_ITEM(apart, i), "ii", &one, &two)) return -1;
        fits = fits && one >= 0 && two >= 0 && one < count && two < count && !plan->planes[one].value && !plan->planes[two].value;
        plan->apart.emplace_back(one, two);
    }
    if (!fits) {
        PyErr_SetString(PyExc_ValueError, "a word past the job's, or a plane that is not there");
        return -1;
    }
    return 0;
}

void call_dealloc(PyObject* self) {
    PyTypeObject* type = Py_TYPE(self);
    if (Plan* plan = reinterpret_cast<Call*>(self)->plan) {
        for (Plane& p : plan->planes) Py_DECREF(p.name);
        delete plan;
    }
    type->tp_free(self);
    Py_DECREF(type);
}

bool address_of(const Plan& plan, const Plane& p, PyObject* x, uint64_t& at) {
    if (!THPVariable_CheckExact(x)) return false;
    const at::Tensor& t = THPVariable_Unpack(x);
    if (t.scalar_type() != p.type || !t.is_cuda() || t.get_device() != plan.device || t.sizes() != at::IntArrayRef(p.sizes) ||
        t.strides() != at::IntArrayRef(p.strides))
        return false;
    at = reinterpret_cast<uint64_t>(t.data_ptr());
    return true;
}

// run(arrays, device, stream): the entry's status, or -1 for a call that is not the
// plan's (other planes, a stream without its space or under capture, whose space is
// the graph's), of which nothing ran.
PyObject* call_run(PyObject* self, PyObject* const* args, Py_ssize_t n) {
    if (n != 3 || !PyDict_CheckExact(args[0])) {
        PyErr_SetString(PyExc_TypeError, "run(arrays, device, stream)");
        return nullptr;
    }
    const Plan& plan = *reinterpret_cast<Call*>(self)->plan;
    const long device = PyLong_AsLong(args[1]);
    const uint64_t stream = PyLong_AsUnsignedLongLong(args[2]);
    if (PyErr_Occurred()) return nullptr;
    const size_t count = plan.planes.size();
    if (device != plan.device || static_cast<size_t>(PyDict_GET_SIZE(args[0])) != count) return PyLong_FromLong(-1);
    uint64_t job[kMostWords];
    std::memcpy(job, plan.job.data(), 8 * plan.job.size());
    uint64_t at[kMostWords];
    if (count > kMostWords) return PyLong_FromLong(-1);
    PyObject *name, *x;
    Py_ssize_t where = 0;
    try {
        for (size_t i = 0; PyDict_Next(args[0], &where, &name, &x); ++i) {
            const Plane& p = plan.planes[i];
            if (name != p.name) return PyLong_FromLong(-1);
            at[i] = 0;
            if (p.value) {
                if (!PyLong_CheckExact(x)) return PyLong_FromLong(-1);
                at[i] = PyLong_AsUnsignedLongLong(x);
                if (at[i] == ~0ull && PyErr_Occurred()) {
                    PyErr_Clear();
                    return PyLong_FromLong(-1);
                }
            } else if (!address_of(plan, p, x, at[i])) {
                return PyLong_FromLong(-1);
            }
            if (p.word >= 0) job[p.word] = at[i];
        }
    } catch (const std::exception&) {       // a tensor without strides or memory
        return PyLong_FromLong(-1);
    }
    for (const auto& pair : plan.apart)
        if (at[pair.first] == at[pair.second]) return PyLong_FromLong(-1);
    uint64_t scratch = 0;
    std::mutex* launches = nullptr;
    if (plan.needs_space) {
        const Space* space = nullptr;
        for (const Space& s : plan.spaces)
            if (s.stream == stream) space = &s;
        if (!space || (plan.capturing && plan.capturing(reinterpret_cast<void*>(stream)))) return PyLong_FromLong(-1);
        scratch = space->scratch;
        launches = space->launches;
        if (plan.state_word >= 0) job[plan.state_word] = space->state;
    }
    return PyLong_FromLong(enter(plan, job, scratch, stream, launches));
}

// launch(bound, scratch, stream): the entry's status with the words of `bound`, a
// list of (word, value), put into the job.
PyObject* call_launch(PyObject* self, PyObject* args) {
    PyObject* bound;
    unsigned long long scratch, stream;
    if (!PyArg_ParseTuple(args, "O!KK", &PyList_Type, &bound, &scratch, &stream)) return nullptr;
    const Plan& plan = *reinterpret_cast<Call*>(self)->plan;
    uint64_t job[kMostWords];
    std::memcpy(job, plan.job.data(), 8 * plan.job.size());
    for (Py_ssize_t i = 0; i < PyList_GET_SIZE(bound); ++i) {
        long long word;
        unsigned long long value;
        if (!PyArg_ParseTuple(PyList_GET_ITEM(bound, i), "LK", &word, &value)) return nullptr;
        if (word < 0 || static_cast<size_t>(word) >= plan.job.size()) {
            PyErr_SetString(PyExc_ValueError, "a word past the job's");
            return nullptr;
        }
        job[word] = value;
    }
    return PyLong_FromLong(enter(plan, job, scratch, stream, plan.needs_space ? launches_of(plan.device, stream) : nullptr));
}

// space(stream, scratch, state): what the calls on a stream work in.
PyObject* call_space(PyObject* self, PyObject* args) {
    unsigned long long stream, scratch, state;
    if (!PyArg_ParseTuple(args, "KKK", &stream, &scratch, &state)) return nullptr;
    Plan& plan = *reinterpret_cast<Call*>(self)->plan;
    plan.spaces.push_back({stream, scratch, state, launches_of(plan.device, stream)});
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"run", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(call_run)), METH_FASTCALL, nullptr},
    {"launch", call_launch, METH_VARARGS, nullptr},
    {"space", call_space, METH_VARARGS, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyType_Slot slots[] = {
    {Py_tp_init, reinterpret_cast<void*>(call_init)},
    {Py_tp_new, reinterpret_cast<void*>(PyType_GenericNew)},
    {Py_tp_dealloc, reinterpret_cast<void*>(call_dealloc)},
    {Py_tp_methods, methods},
    {0, nullptr},
};
PyType_Spec spec = {"hawk_amd._bind.Call", sizeof(Call), 0, Py_TPFLAGS_DEFAULT, slots};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_bind", nullptr, -1, nullptr, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__bind(void) {
    PyObject* made = PyModule_Create(&module);
    PyObject* type = made ? PyType_FromSpec(&spec) : nullptr;
    if (!type || PyModule_AddObject(made, "Call", type) < 0 || PyModule_AddStringConstant(made, "digest", HAWK_BUILD_DIGEST) < 0)
        return nullptr;
    return made;
}
