// gs_host.cpp -- argument checks, address columns and the library calls of the operators on lists of tensors (optim.py), as a
// CPython module.
//
// A step of 180 tensors looks at five to eight properties of some 900 tensor objects.  Python spends 0.3 us on each object
// (0.25 ms a step, as long as the kernels run); reading the same fields from C++ takes 0.03 us, and a call
// of twenty arguments 0.1 us where ctypes takes 3.  The module keeps nothing between calls but the library's addresses.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <c10/core/ScalarType.h>
#include <torch/csrc/autograd/python_variable.h>

#include <string>
#include <vector>

#include "../../include/gsplat_hip.h"

namespace {

constexpr int64_t BLOCK = 64;       // elements that share the exponents of 8-bit moments where blocks are not rows

// What a list of a call holds; the first list of a call is the one whose shapes the others have.
enum Kind {
    PARAM = 0,      // float32, bfloat16 or float16, contiguous                              (first list)
    GRAD = 1,       // the type of the first list's tensor; copied where it is not contiguous
    GRADS = 2,      // float32, bfloat16 or float16; copied where it is not contiguous        (first list)
    FLOAT = 3,      // float32
    MASTER = 4,     // float32 or None; a float32 parameter has none
    CODE = 5,       // uint8                                                                  (first list, too)
    EXPONENTS = 6,  // uint8 [blocks, 2]
    MASK = 7,       // int8 [rows] or None
    PARAM_MASK = 8, // the same, of a float32 parameter
    STAMP = 9,      // int32 [rows], None where the list before has None
    VALUE = 10,     // all float32 or all bfloat16
};

int dtype_code(at::ScalarType t) { return t == at::kFloat ? 0 : t == at::kBFloat16 ? 1 : t == at::kHalf ? 2 : -1; }

int64_t row_length(c10::IntArrayRef s) { return s.size() == 2 && s[1] >= 1 && s[1] <= BLOCK ? s[1] : 0; }
int64_t num_blocks(c10::IntArrayRef s, int64_t numel) { return row_length(s) ? s[0] : (numel + BLOCK - 1) / BLOCK; }

std::string shape_text(c10::IntArrayRef s) {
    std::string t = "(";
    for (size_t i = 0; i < s.size(); ++i) t += (i ? ", " : "") + std::to_string(s[i]);
    return t + (s.size() == 1 ? ",)" : ")");
}

struct Refused {
    PyObject *type;
    std::string text;
};

std::string at_place(const char *name, Py_ssize_t i) { return std::string(name) + "[" + std::to_string(i) + "]"; }

struct Holder {     // a reference that ends with its scope
    PyObject *o;
    explicit Holder(PyObject *p) : o(p) {}
    ~Holder() { Py_XDECREF(o); }
    Holder(const Holder &) = delete;
};

PyObject *column_bytes(const void *data, size_t bytes) { return PyBytes_FromStringAndSize((const char *)data, (Py_ssize_t)bytes); }

// collect(lists): lists = ((name, sequence or None, kind), ...).  Returns (columns, numel, rows, dtypes, device index, kept):
// address columns (bytes of uint64, None for a list that is None), the first list's element counts (int64), row lengths
// (int32) and type codes (int32), and the contiguous copies that have to live until the kernels are enqueued.
PyObject *collect_checked(PyObject *lists) {
    const Py_ssize_t n_lists = PyTuple_GET_SIZE(lists);
    Holder columns(PyTuple_New(n_lists)), kept(PyList_New(0));
    if (!columns.o || !kept.o) return nullptr;
    std::vector<const at::Tensor *> first;
    std::vector<int64_t> numel;
    std::vector<int32_t> rows, types;
    std::vector<uint64_t> address;
    std::vector<char> given;        // of the last list
    struct List { const char *name; PyObject *fast; int kind; };     // (fast: null for None; `kept` holds the references)
    std::vector<List> all(n_lists);
    Py_ssize_t n = 0;
    for (Py_ssize_t k = 0; k < n_lists; ++k) {
        PyObject *name_object, *values;
        if (!PyArg_ParseTuple(PyTuple_GET_ITEM(lists, k), "UOi", &name_object, &values, &all[k].kind)) return nullptr;
        all[k].name = PyUnicode_AsUTF8(name_object);
        all[k].fast = nullptr;
        if (values == Py_None && k > 0) continue;
        Holder fast(PySequence_Fast(values, "a sequence of tensors"));
        if (!fast.o || PyList_Append(kept.o, fast.o) < 0) return nullptr;
        all[k].fast = fast.o;
        const Py_ssize_t length = PySequence_Fast_GET_SIZE(fast.o);
        if (k == 0) n = length;
        else if (length != n)
            throw Refused{PyExc_ValueError, std::string(all[k].name) + ": " + std::to_string(length) + " entries for " + std::to_string(n) + " tensors"};
    }
    first.resize(n);
    numel.resize(n);
    rows.resize(n);
    types.resize(n);
    int device = -1;
    for (Py_ssize_t k = 0; k < n_lists; ++k) {
        const char *name = all[k].name;
        const int kind = all[k].kind;
        if (!all[k].fast) {
            Py_INCREF(Py_None);
            PyTuple_SET_ITEM(columns.o, k, Py_None);
            given.clear();
            continue;
        }
        address.assign(n, 0);
        std::vector<char> before;
        before.swap(given);
        given.assign(n, 0);
        at::ScalarType value_type = at::kFloat;
        for (Py_ssize_t i = 0; i < n; ++i) {
            PyObject *o = PySequence_Fast_GET_ITEM(all[k].fast, i);
            if (o == Py_None && (kind == MASTER || kind == MASK || kind == PARAM_MASK || kind == STAMP)) {
                if (kind == STAMP && !before.empty() && before[i])
                    throw Refused{PyExc_ValueError, at_place(name, i) + ": row masks and last steps come together"};
                continue;
            }
            if (!THPVariable_Check(o)) throw Refused{PyExc_TypeError, at_place(name, i) + " is no tensor"};
            const at::Tensor &t = THPVariable_Unpack(o);
            given[i] = 1;
            if (t.layout() != at::kStrided) throw Refused{PyExc_RuntimeError, at_place(name, i) + " is sparse: dense tensors are taken"};
            if (!t.is_cuda()) throw Refused{PyExc_RuntimeError, at_place(name, i) + " is on " + t.device().str() + ", not on the HIP device: there is no CPU path"};
            if (device < 0) device = t.device().index();
            if (t.device().index() != device)
                throw Refused{PyExc_RuntimeError, at_place(name, i) + " is on " + t.device().str() + ": all tensors of a call belong on one HIP device"};
            const at::ScalarType type = t.scalar_type();
            if (k == 0) {
                first[i] = &t;
                numel[i] = t.numel();
                rows[i] = (int32_t)row_length(t.sizes());
                types[i] = dtype_code(type);
            }
            const at::Tensor &ref = *first[i];
            bool right_type = true;
            if (kind == PARAM || kind == GRADS) right_type = types[i] >= 0;
            else if (kind == GRAD) right_type = type == ref.scalar_type();
            else if (kind == FLOAT || kind == MASTER) right_type = type == at::kFloat;
            else if (kind == CODE || kind == EXPONENTS) right_type = type == at::kByte;
            else if (kind == MASK || kind == PARAM_MASK) right_type = type == at::kChar;
            else if (kind == STAMP) right_type = type == at::kInt;
            else if (kind == VALUE) {
                if (i == 0) value_type = type;
                right_type = type == value_type && (type == at::kFloat || type == at::kBFloat16);
            }
            if (!right_type)
                throw Refused{PyExc_TypeError, at_place(name, i) + " is of type " + c10::toString(type) +
                                                   (kind == PARAM || kind == GRADS ? ": float32, bfloat16 and float16 are supported" : ", which this list does not take")};
            if (kind == MASTER && ref.scalar_type() == at::kFloat)
                throw Refused{PyExc_ValueError, at_place(name, i) + ": a float32 parameter is its own master copy"};
            if (kind == STAMP && !before.empty() && !before[i])
                throw Refused{PyExc_ValueError, at_place(name, i) + ": row masks and last steps come together"};
            if ((kind == MASK || kind == PARAM_MASK) && rows[i] == 0)
                throw Refused{PyExc_ValueError, at_place(name, i) + ": the tensor has no rows of 1 to " + std::to_string(BLOCK) + " elements"};
            if (kind == PARAM_MASK && ref.scalar_type() != at::kFloat)
                throw Refused{PyExc_TypeError, at_place(name, i) + ": row masks are for float32 parameters"};
            bool right_shape;
            if (kind == EXPONENTS) right_shape = t.dim() == 2 && t.size(0) == num_blocks(ref.sizes(), numel[i]) && t.size(1) == 2;
            else if (kind == MASK || kind == PARAM_MASK || kind == STAMP) right_shape = t.dim() == 1 && t.size(0) == ref.size(0);
            else right_shape = k == 0 || t.sizes() == ref.sizes();
            if (!right_shape)
                throw Refused{PyExc_ValueError, at_place(name, i) + " has shape " + shape_text(t.sizes()) + ", which does not fit a tensor of shape " + shape_text(ref.sizes())};
            if (t.is_contiguous() && !t.is_neg()) {
                address[i] = (uint64_t)(uintptr_t)t.const_data_ptr();
            } else if (kind == GRAD || kind == GRADS) {
                const at::Tensor copy = t.detach().resolve_neg().contiguous();
                Holder wrapped(THPVariable_Wrap(copy));
                if (!wrapped.o || PyList_Append(kept.o, wrapped.o) < 0) return nullptr;
                address[i] = (uint64_t)(uintptr_t)copy.const_data_ptr();
            } else {
                throw Refused{PyExc_ValueError, at_place(name, i) + " is not contiguous"};
            }
        }
        PyObject *column = column_bytes(address.data(), address.size() * 8);
        if (!column) return nullptr;
        PyTuple_SET_ITEM(columns.o, k, column);
    }
    Holder a(column_bytes(numel.data(), numel.size() * 8)), b(column_bytes(rows.data(), rows.size() * 4)), c(column_bytes(types.data(), types.size() * 4));
    if (!a.o || !b.o || !c.o) return nullptr;
    return Py_BuildValue("(OOOOiO)", columns.o, a.o, b.o, c.o, device, kept.o);
}

// One value for all tensors, or a list or tuple with one for each: the object for tensor i (borrowed)
struct PerTensor {
    PyObject *values;
    bool list;
    PerTensor(const char *name, PyObject *v, Py_ssize_t n) : values(v), list(PyList_Check(v) || PyTuple_Check(v)) {
        if (list && PySequence_Fast_GET_SIZE(v) != n)
            throw Refused{PyExc_ValueError, std::string(name) + ": " + std::to_string(PySequence_Fast_GET_SIZE(v)) + " entries for " + std::to_string(n) + " tensors"};
    }
    PyObject *operator[](Py_ssize_t i) const { return list ? PySequence_Fast_GET_ITEM(values, i) : values; }
};

const at::Tensor *device_scalar(const char *name, Py_ssize_t i, PyObject *o, at::ScalarType type, int device) {
    if (!THPVariable_Check(o)) return nullptr;
    const at::Tensor &t = THPVariable_Unpack(o);
    if (!t.is_cuda() || t.device().index() != device || t.scalar_type() != type || t.numel() != 1)
        throw Refused{PyExc_ValueError, at_place(name, i) + ": a number, or one " + c10::toString(type) + " on the parameters' device"};
    return &t;
}

// scalars(n, step, lr, weight_decay, beta1, beta2, eps, device): each of the first three for all tensors or one per tensor;
// step and lr may be device tensors.  Returns (hyper float64 [n][5], counts int64 [n], step addresses or None, lr addresses or
// None, whether any step is a number).
PyObject *scalars_checked(PyObject *args) {
    Py_ssize_t n;
    PyObject *step, *lr, *decay;
    double beta1, beta2, eps;
    int device;
    if (!PyArg_ParseTuple(args, "nOOOdddi", &n, &step, &lr, &decay, &beta1, &beta2, &eps, &device)) return nullptr;
    const PerTensor steps("step", step, n), rates("lr", lr, n), decays("weight_decay", decay, n);
    std::vector<double> hyper((size_t)n * 5);
    std::vector<int64_t> counts(n, 0);
    std::vector<uint64_t> step_at(n, 0), rate_at(n, 0);
    bool step_tensor = false, rate_tensor = false, number = false;
    for (Py_ssize_t i = 0; i < n; ++i) {
        if (const at::Tensor *t = device_scalar("step", i, steps[i], at::kLong, device)) {
            step_at[i] = (uint64_t)(uintptr_t)t->const_data_ptr();
            step_tensor = true;
        } else {
            counts[i] = PyLong_AsLongLong(steps[i]);
            if (counts[i] == -1 && PyErr_Occurred()) return nullptr;
            if (counts[i] < 1) throw Refused{PyExc_ValueError, "step counts from 1"};
            number = true;
        }
        double *h = &hyper[(size_t)i * 5];
        if (const at::Tensor *t = device_scalar("lr", i, rates[i], at::kFloat, device)) {
            rate_at[i] = (uint64_t)(uintptr_t)t->const_data_ptr();
            rate_tensor = true;
            h[0] = 0.0;
        } else {
            h[0] = PyFloat_AsDouble(rates[i]);
            if (h[0] == -1.0 && PyErr_Occurred()) return nullptr;
        }
        h[1] = beta1;
        h[2] = beta2;
        h[3] = eps;
        h[4] = PyFloat_AsDouble(decays[i]);
        if (h[4] == -1.0 && PyErr_Occurred()) return nullptr;
        if (!(h[0] >= 0.0) || !(h[4] >= 0.0)) throw Refused{PyExc_ValueError, "invalid AdamW hyper-parameters: lr and weight_decay are at least 0"};
    }
    Holder a(column_bytes(hyper.data(), hyper.size() * 8)), b(column_bytes(counts.data(), counts.size() * 8));
    Holder c(step_tensor ? column_bytes(step_at.data(), step_at.size() * 8) : (Py_INCREF(Py_None), Py_None));
    Holder d(rate_tensor ? column_bytes(rate_at.data(), rate_at.size() * 8) : (Py_INCREF(Py_None), Py_None));
    if (!a.o || !b.o || !c.o || !d.o) return nullptr;
    return Py_BuildValue("(OOOOO)", a.o, b.o, c.o, d.o, number ? Py_True : Py_False);
}

// The library's entry points: it is loaded by the package (which checks its version), not linked here.
decltype(&gs_adamw_step) adamw_step = nullptr;
decltype(&gs_grad_norm) grad_norm = nullptr;
decltype(&gs_read_moments) read_moments = nullptr;

PyObject *bind(PyObject *args) {
    unsigned long long a, b, c;
    if (!PyArg_ParseTuple(args, "KKK", &a, &b, &c)) return nullptr;
    adamw_step = reinterpret_cast<decltype(adamw_step)>(a);
    grad_norm = reinterpret_cast<decltype(grad_norm)>(b);
    read_moments = reinterpret_cast<decltype(read_moments)>(c);
    Py_RETURN_NONE;
}

// The data of a column (bytes), null for None
template <typename T>
const T *column(PyObject *o) {
    if (o == Py_None) return nullptr;
    if (!PyBytes_Check(o)) throw Refused{PyExc_TypeError, "a column of collect() or scalars()"};
    return reinterpret_cast<const T *>(PyBytes_AS_STRING(o));
}
template <typename T>
const T *column(PyObject *tuple, Py_ssize_t i) { return column<T>(PyTuple_GET_ITEM(tuple, i)); }

PyObject *tuple_of(PyObject *o, Py_ssize_t n) {
    if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) < n) throw Refused{PyExc_TypeError, "a tuple of collect() or scalars()"};
    return o;
}

// A graph that has kept one of these tensors for its backward pass must notice that it changed, as after any operation in place.
void count_as_changed(PyObject *tensors) {
    for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(tensors); ++i) {
        PyObject *t = PySequence_Fast_GET_ITEM(tensors, i);
        if (THPVariable_Check(t) && !THPVariable_Unpack(t).is_inference()) THPVariable_Unpack(t).unsafeGetTensorImpl()->bump_version();
    }
}

// step(collected, scalars, ids or None, grad scale address, seed, workspace address, stream): status of gs_adamw_step.
// `collected`: params, grads, exp_avgs, exp_avg_sqs, exponents, masters, row masks, last steps.
PyObject *step(PyObject *args) {
    PyObject *collected, *numbers, *ids;
    unsigned long long scale, workspace, stream;
    unsigned int seed;
    if (!PyArg_ParseTuple(args, "OOOKIKK", &collected, &numbers, &ids, &scale, &seed, &workspace, &stream)) return nullptr;
    PyObject *c = tuple_of(PyTuple_GET_ITEM(tuple_of(collected, 6), 0), 8);
    tuple_of(numbers, 4);
    const Py_ssize_t n = PyBytes_GET_SIZE(PyTuple_GET_ITEM(collected, 1)) / 8;
    std::vector<int32_t> id(n);
    if (ids != Py_None) {
        Holder fast(PySequence_Fast(ids, "tensor_ids: a sequence of numbers"));
        if (!fast.o) return nullptr;
        if (PySequence_Fast_GET_SIZE(fast.o) != n) throw Refused{PyExc_ValueError, "tensor_ids: one for each tensor"};
        for (Py_ssize_t i = 0; i < n; ++i) {
            id[i] = (int32_t)PyLong_AsLong(PySequence_Fast_GET_ITEM(fast.o, i));
            if (id[i] == -1 && PyErr_Occurred()) return nullptr;
        }
    } else {
        for (Py_ssize_t i = 0; i < n; ++i) id[i] = (int32_t)i;
    }
    if (!adamw_step) throw Refused{PyExc_RuntimeError, "the library is not bound"};
    typedef uint64_t U;
    const int status = adamw_step((int)n, column<U>(c, 0), column<U>(c, 1), column<U>(c, 2), column<U>(c, 3), column<U>(c, 4), column<U>(c, 5),
                                  column<U>(c, 6), column<U>(c, 7), column<int64_t>(collected, 1), column<int32_t>(collected, 2), column<int32_t>(collected, 3),
                                  id.data(), column<double>(numbers, 0), column<int64_t>(numbers, 1), column<U>(numbers, 2), column<U>(numbers, 3),
                                  (const float *)scale, seed, (void *)workspace, (void *)stream);
    if (status == 0) count_as_changed(PyList_GET_ITEM(PyTuple_GET_ITEM(collected, 5), 0));
    return PyLong_FromLong(status);
}

// norm(grads column, row mask column, collected, max_norm, sq_sum, norm, clip, each or 0, workspace, stream): status of gs_grad_norm
PyObject *norm(PyObject *args) {
    PyObject *grads, *masks, *collected;
    double max_norm;
    unsigned long long sq_sum, total, clip, each, workspace, stream;
    if (!PyArg_ParseTuple(args, "OOOdKKKKKK", &grads, &masks, &collected, &max_norm, &sq_sum, &total, &clip, &each, &workspace, &stream)) return nullptr;
    tuple_of(collected, 4);
    if (!grad_norm) throw Refused{PyExc_RuntimeError, "the library is not bound"};
    return PyLong_FromLong(grad_norm((int)(PyBytes_GET_SIZE(PyTuple_GET_ITEM(collected, 1)) / 8), column<uint64_t>(grads), column<uint64_t>(masks),
                                     column<int64_t>(collected, 1), column<int32_t>(collected, 2), column<int32_t>(collected, 3), max_norm, (double *)sq_sum,
                                     (float *)total, (float *)clip, (float *)each, (void *)workspace, (void *)stream));
}

// read(collected, type code, stream): status of gs_read_moments.  `collected`: exp_avgs, exp_avg_sqs, exponents and the two outputs.
PyObject *read(PyObject *args) {
    PyObject *collected;
    int dtype;
    unsigned long long stream;
    if (!PyArg_ParseTuple(args, "OiK", &collected, &dtype, &stream)) return nullptr;
    PyObject *c = tuple_of(PyTuple_GET_ITEM(tuple_of(collected, 6), 0), 5);
    if (!read_moments) throw Refused{PyExc_RuntimeError, "the library is not bound"};
    typedef uint64_t U;
    const int status = read_moments((int)(PyBytes_GET_SIZE(PyTuple_GET_ITEM(collected, 1)) / 8), column<U>(c, 0), column<U>(c, 1), column<U>(c, 2),
                                    column<U>(c, 3), column<U>(c, 4), column<int64_t>(collected, 1), column<int32_t>(collected, 2), dtype, (void *)stream);
    PyObject *kept = PyTuple_GET_ITEM(collected, 5);        // (the five lists, in their order)
    for (Py_ssize_t k = 3; status == 0 && k < 5; ++k) count_as_changed(PyList_GET_ITEM(kept, k));
    return PyLong_FromLong(status);
}

template <PyObject *(*F)(PyObject *)>
PyObject *guarded(PyObject *, PyObject *args) {
    try {
        return F(args);
    } catch (const Refused &r) {
        PyErr_SetString(r.type, r.text.c_str());
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

PyMethodDef methods[] = {
    {"collect", guarded<collect_checked>, METH_VARARGS, "collect((name, tensors or None, kind), ...): checked address columns"},
    {"scalars", guarded<scalars_checked>, METH_VARARGS, "scalars(n, step, lr, weight_decay, beta1, beta2, eps, device): checked number columns"},
    {"bind", guarded<bind>, METH_VARARGS, "bind(gs_adamw_step, gs_grad_norm, gs_read_moments): the library's addresses"},
    {"step", guarded<step>, METH_VARARGS, "gs_adamw_step on collected columns"},
    {"norm", guarded<norm>, METH_VARARGS, "gs_grad_norm on collected columns"},
    {"read", guarded<read>, METH_VARARGS, "gs_read_moments on collected columns"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_gs_host", "argument columns of the operators on lists of tensors", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__gs_host(void) {
    PyObject *m = PyModule_Create(&module_def);
    if (!m) return nullptr;
    const struct { const char *name; int value; } kinds[] = {{"PARAM", PARAM}, {"GRAD", GRAD}, {"GRADS", GRADS}, {"FLOAT", FLOAT}, {"MASTER", MASTER},
        {"CODE", CODE}, {"EXPONENTS", EXPONENTS}, {"MASK", MASK}, {"PARAM_MASK", PARAM_MASK}, {"STAMP", STAMP}, {"VALUE", VALUE}};
    for (const auto &k : kinds)
        if (PyModule_AddIntConstant(m, k.name, k.value) < 0) return nullptr;
    // (of the header that the calls above were compiled from: the package compares it with the library's before it binds)
    if (PyModule_AddIntConstant(m, "ABI_VERSION", GS_ABI_VERSION) < 0) return nullptr;
    return m;
}
