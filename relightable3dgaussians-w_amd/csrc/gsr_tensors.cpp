// gsr_tensors.cpp -- what an optimizer step asks of a list of torch tensors, in one call (host only,
// libgsr_tensors.so; called through ctypes.PyDLL with the interpreter's lock held).
//
// A step over n parameters looks at n gradients, n parameters and 3 to 6 n state tensors: their
// addresses, sizes, types and devices.  From Python each look is a method call of 35 to 50 ns, about
// 0.8 us a parameter (300 parameters: 230 us, as long as the GPU takes for 63M elements); here one is
// 5 to 20 ns.  Nothing is launched, kept or changed; libgsr.so stays free of torch.
#include <ATen/Functions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <utility>
#include <vector>

#include "../../include/gsr.h"

namespace {

// What a tensor is, in five words: address, elements, type (gsr.h's 0, 1, 2; 3 e4m3, 4 int64, -1 another,
// -2 None, -3 no tensor), device (-1: not a GPU), dense (contiguous, strided,
// its memory holding its values and not their negatives)
constexpr int WORDS = 5;

void describe(PyObject* o, long long* out) {
    out[0] = out[1] = out[4] = 0;
    out[3] = -1;
    if (o == nullptr || o == Py_None) {
        out[2] = -2;
        return;
    }
    if (!THPVariable_Check(o)) {
        out[2] = -3;
        return;
    }
    const at::Tensor& t = THPVariable_Unpack(o);
    const at::ScalarType s = t.scalar_type();
    out[1] = t.numel();
    out[2] = s == at::kFloat ? 0 : s == at::kBFloat16 ? 1 : s == at::kHalf ? 2 : s == at::kFloat8_e4m3fn ? 3 : s == at::kLong ? 4 : -1;
    if (t.layout() != at::kStrided) return;
    out[0] = (long long)reinterpret_cast<uintptr_t>(t.data_ptr());
    out[3] = t.is_cuda() ? t.device().index() : -1;
    out[4] = t.is_contiguous() && !t.is_neg();
}

bool same(PyObject* o, const long long* expected) {
    long long now[WORDS];
    describe(o, now);
    for (int k = 0; k < WORDS; k++)
        if (now[k] != expected[k]) return false;
    return true;
}

// Runs f, whose torch calls may throw (a tensor without storage): nothing leaves a C entry that way
template <typename F>
auto guarded(F f, decltype(f()) failed) -> decltype(f()) {
    try {
        return f();
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "gsr_tensors: unknown error");
    }
    return failed;
}

// Pieces of memory, those of nothing left out
struct Spans {
    std::vector<std::pair<uintptr_t, uintptr_t>> v;  // [begin, end)
    void add(const void* p, long long bytes) {
        const uintptr_t at = reinterpret_cast<uintptr_t>(p);
        if (bytes > 0) v.emplace_back(at, at + (uintptr_t)bytes);
    }
    int overlap() {
        std::sort(v.begin(), v.end());
        for (size_t i = 1; i < v.size(); i++)
            if (v[i].first < v[i - 1].second) return 1;
        return 0;
    }
};

}  // namespace

extern "C" {

// WORDS words of each of a list's items; 0, or -1 if it is no list
int gsr_tensors_describe(PyObject* list, long long* out) {
    return guarded(
        [&] {
            if (!PyList_Check(list)) return -1;
            for (Py_ssize_t i = 0; i < PyList_GET_SIZE(list); i++) describe(PyList_GET_ITEM(list, i), out + WORDS * i);
            return 0;
        },
        -1);
}

// The same of each of `names` (a tuple) in each of a list of dicts, one dict after another
int gsr_tensors_describe_states(PyObject* states, PyObject* names, long long* out) {
    return guarded(
        [&] {
            if (!PyList_Check(states) || !PyTuple_Check(names)) return -1;
            for (Py_ssize_t i = 0; i < PyList_GET_SIZE(states); i++) {
                PyObject* st = PyList_GET_ITEM(states, i);
                if (!PyDict_Check(st)) return -1;
                for (Py_ssize_t k = 0; k < PyTuple_GET_SIZE(names); k++, out += WORDS)
                    describe(PyDict_GetItem(st, PyTuple_GET_ITEM(names, k)), out);
            }
            return 0;
        },
        -1);
}

// The gradients of a list of parameters that have one, as a new list
PyObject* gsr_tensors_grads(PyObject* params) {
    return guarded(
        [&]() -> PyObject* {
            PyObject* out = PyList_New(0);
            if (out == nullptr) return nullptr;
            for (Py_ssize_t i = 0; i < PyList_GET_SIZE(params); i++) {
                PyObject* p = PyList_GET_ITEM(params, i);
                if (!THPVariable_Check(p)) {
                    PyErr_SetString(PyExc_TypeError, "a parameter is not a tensor");
                    Py_DECREF(out);
                    return nullptr;
                }
                const at::Tensor& g = THPVariable_Unpack(p).grad();
                if (!g.defined()) continue;
                PyObject* o = THPVariable_Wrap(g);
                if (o == nullptr || PyList_Append(out, o) != 0) {
                    Py_XDECREF(o);
                    Py_DECREF(out);
                    return nullptr;
                }
                Py_DECREF(o);
            }
            return out;
        },
        nullptr);
}

// The table that gsr_grad_norm takes of a list of gradients: their device, or -1 where one is no dense
// float, bfloat16 or half tensor of one GPU
int gsr_tensors_grad_table(PyObject* grads, gsr_grad_tensor* out) {
    return guarded(
        [&] {
            int device = -1;
            for (Py_ssize_t i = 0; i < PyList_GET_SIZE(grads); i++, out++) {
                long long w[WORDS];
                describe(PyList_GET_ITEM(grads, i), w);
                if (w[2] < 0 || w[2] > 2 || w[3] < 0 || !w[4] || (i && w[3] != device)) return -1;
                device = (int)w[3];
                out->grad = reinterpret_cast<void*>((uintptr_t)w[0]);
                out->n = w[1];
                out->type = (int)w[2];
                out->reserved = 0;
            }
            return device;
        },
        -1);
}

// Whether two of a table's gradients share memory: 1, 0, or -1
int gsr_tensors_overlap(const gsr_grad_tensor* t, int count) {
    return guarded(
        [&] {
            Spans spans;
            for (int i = 0; i < count; i++) spans.add(t[i].grad, t[i].n * (t[i].type == 0 ? 4 : 2));
            return spans.overlap();
        },
        -1);
}

// The table that gsr_adamw_step takes, but for gradients, rates and step counts on the host: params with
// their states (dicts of `names`: exp_avg, exp_avg_sq and, of moments in 8 bits, their scales, master, step),
// which are to be on GPU `device`; places: the ordinals.  0, or 1 where a tensor is not what it should be.
int gsr_tensors_plan(PyObject* params, PyObject* states, PyObject* names, int bits, int counted, int device,
                     const int* places, gsr_adamw_tensor* out) {
    return guarded(
        [&] {
            const int moments = bits == 8 ? 4 : 2, codes = bits == 8 ? 3 : 0;
            for (Py_ssize_t i = 0; i < PyList_GET_SIZE(params); i++) {
                PyObject* st = PyList_GET_ITEM(states, i);
                if (!PyDict_Check(st) || PyTuple_GET_SIZE(names) != moments + 2) return 1;
                long long p[WORDS], w[6][WORDS];
                describe(PyList_GET_ITEM(params, i), p);
                for (int k = 0; k < moments + 2; k++) describe(PyDict_GetItem(st, PyTuple_GET_ITEM(names, k)), w[k]);
                auto good = [&](const long long* x, int type, long long n) {
                    return x[2] == type && x[1] == n && x[3] == device && x[4];
                };
                if (p[2] < 0 || p[2] > 2 || p[3] != device || !p[4]) return 1;
                for (int k = 0; k < 2; k++)
                    if (!good(w[k], codes, p[1]) || (bits == 8 && !good(w[2 + k], 0, (p[1] + 255) / 256))) return 1;
                if ((p[2] && !good(w[moments], 0, p[1])) || (counted && !good(w[moments + 1], 4, 1))) return 1;
                auto at = [](const long long* x) { return reinterpret_cast<void*>((uintptr_t)x[0]); };
                gsr_adamw_tensor& t = out[i];
                t = gsr_adamw_tensor{};
                t.param = at(p);
                t.n = p[1];
                t.param_type = (int)p[2];
                t.exp_avg = at(w[0]);
                t.exp_avg_sq = at(w[1]);
                if (bits == 8) {
                    t.exp_avg_scale = static_cast<float*>(at(w[2]));
                    t.exp_avg_sq_scale = static_cast<float*>(at(w[3]));
                }
                if (p[2]) t.master = static_cast<float*>(at(w[moments]));
                if (counted) t.step_dev = static_cast<long long*>(at(w[moments + 1]));
                t.step = 1;
                t.ordinal = places[i];
            }
            return 0;
        },
        -1);
}

// Whether what a step over the table writes overlaps: 1, 0, or -1
int gsr_tensors_written_overlap(const gsr_adamw_tensor* t, int count, int bits) {
    return guarded(
        [&] {
            Spans spans;
            for (int i = 0; i < count; i++) {
                const long long n = t[i].n, moment = bits == 8 ? n : 4 * n, scales = 4 * ((n + 255) / 256);
                spans.add(t[i].param, n * (t[i].param_type == 0 ? 4 : 2));
                spans.add(t[i].exp_avg, moment);
                spans.add(t[i].exp_avg_sq, moment);
                if (t[i].master) spans.add(t[i].master, 4 * n);
                if (bits == 8) {
                    spans.add(t[i].exp_avg_scale, scales);
                    spans.add(t[i].exp_avg_sq_scale, scales);
                }
                if (t[i].step_dev) spans.add(t[i].step_dev, 8);
            }
            return spans.overlap();
        },
        -1);
}

// Selections of rows of 8-bit moments.  `tensors`, five for each: the codes and the scales of both moments
// and the index.  Fills the table that gsr_moment_rows takes and returns a new list of four tensors for
// each, room for the rows (the codes of the old ones' shape but for its first dimension, a scale for each
// 256 of them); None where one is not what it should be.
PyObject* gsr_tensors_moment_rows(PyObject* tensors, gsr_moment_rows_tensor* out) {
    return guarded(
        [&]() -> PyObject* {
            const Py_ssize_t n = PyList_GET_SIZE(tensors);
            if (n % 5) Py_RETURN_NONE;
            long long device = -1;
            for (Py_ssize_t i = 0; i < n; i += 5) {
                constexpr long long KINDS[5] = {3, 3, 0, 0, 4};
                long long w[5][WORDS];
                for (int k = 0; k < 5; k++) {
                    describe(PyList_GET_ITEM(tensors, i + k), w[k]);
                    if (w[k][2] != KINDS[k] || w[k][3] < 0 || !w[k][4]) Py_RETURN_NONE;
                    if (i + k == 0) device = w[k][3];
                    if (w[k][3] != device) Py_RETURN_NONE;
                }
                const at::Tensor& codes = THPVariable_Unpack(PyList_GET_ITEM(tensors, i));
                const long long blocks = (w[0][1] + 255) / 256;
                if (codes.dim() < 1 || codes.sizes() != THPVariable_Unpack(PyList_GET_ITEM(tensors, i + 1)).sizes() ||
                    w[2][1] != blocks || w[3][1] != blocks || THPVariable_Unpack(PyList_GET_ITEM(tensors, i + 4)).dim() != 1)
                    Py_RETURN_NONE;
                long long cols = 1;
                for (int64_t d : codes.sizes().slice(1)) cols *= d;
                if (cols > 0x7fffffff) {
                    PyErr_Format(PyExc_ValueError, "moments8_rows: rows of %lld elements", cols);
                    return nullptr;
                }
                gsr_moment_rows_tensor& t = out[i / 5];
                t = gsr_moment_rows_tensor{};
                t.src_exp_avg = reinterpret_cast<void*>((uintptr_t)w[0][0]);
                t.src_exp_avg_root = reinterpret_cast<void*>((uintptr_t)w[1][0]);
                t.src_exp_avg_scale = reinterpret_cast<float*>((uintptr_t)w[2][0]);
                t.src_exp_avg_root_scale = reinterpret_cast<float*>((uintptr_t)w[3][0]);
                t.index = reinterpret_cast<long long*>((uintptr_t)w[4][0]);
                t.src_rows = codes.size(0);
                t.rows = cols ? w[4][1] : 0;  // rows of no elements: nothing to move
                t.cols = cols ? (int)cols : 1;
            }
            PyObject* list = PyList_New(n / 5 * 4);
            if (list == nullptr) return nullptr;
            for (Py_ssize_t i = 0; i < n / 5; i++) {
                const at::Tensor& codes = THPVariable_Unpack(PyList_GET_ITEM(tensors, 5 * i));
                c10::SmallVector<int64_t, 5> shape(codes.sizes().begin(), codes.sizes().end());
                shape[0] = THPVariable_Unpack(PyList_GET_ITEM(tensors, 5 * i + 4)).numel();
                const long long blocks = (out[i].rows * out[i].cols + 255) / 256;
                const auto options = at::TensorOptions().device(codes.device());
                gsr_moment_rows_tensor& t = out[i];
                for (int k = 0; k < 4; k++) {
                    at::Tensor x;
                    try {
                        x = k < 2 ? at::empty(shape, options.dtype(at::kFloat8_e4m3fn)) : at::empty({blocks}, options.dtype(at::kFloat));
                    } catch (...) {
                        Py_DECREF(list);
                        throw;
                    }
                    void* to = x.data_ptr();
                    if (k == 0) t.exp_avg = to;
                    if (k == 1) t.exp_avg_root = to;
                    if (k == 2) t.exp_avg_scale = static_cast<float*>(to);
                    if (k == 3) t.exp_avg_root_scale = static_cast<float*>(to);
                    PyObject* o = THPVariable_Wrap(std::move(x));
                    if (o == nullptr) {
                        Py_DECREF(list);
                        return nullptr;
                    }
                    PyList_SET_ITEM(list, 4 * i + k, o);
                }
            }
            return list;
        },
        nullptr);
}

// Whether an optimizer's tensors are those that its tables were made of.
//   groups, params, words:   the param groups' parameters are `params`, each with its WORDS words in `words`
//                            and with or without a gradient as words[WORDS] says (1, 0), WORDS + 2 a row
//   state, keys, values:     the state's keys and dicts are these
//   names, state_words:      and the dicts hold these tensors
// If so a new list of the gradients (or None), with at[i] their addresses, *plain whether each is
// dense, on its parameter's device, as large and of the type words[WORDS + 1], and *written whether a 16-bit
// parameter that has one is of another version than versions[i] (-1: any is right); else None.
PyObject* gsr_tensors_current(PyObject* groups, PyObject* params, const long long* words, PyObject* state, PyObject* keys,
                              PyObject* values, PyObject* names, const long long* state_words, long long* at, int* plain,
                              const long long* versions, int* written) {
    return guarded(
        [&]() -> PyObject* {
            const Py_ssize_t n = PyList_GET_SIZE(params);
            Py_ssize_t i = 0;
            for (Py_ssize_t g = 0; g < PyList_GET_SIZE(groups); g++) {
                PyObject* own = PyDict_GetItemString(PyList_GET_ITEM(groups, g), "params");
                if (own == nullptr || !PyList_Check(own)) Py_RETURN_NONE;
                for (Py_ssize_t k = 0; k < PyList_GET_SIZE(own); k++, i++) {
                    PyObject* p = PyList_GET_ITEM(own, k);
                    if (i >= n || p != PyList_GET_ITEM(params, i) || !same(p, words + (WORDS + 2) * i)) Py_RETURN_NONE;
                }
            }
            if (i != n || !PyDict_Check(state) || PyDict_Size(state) != PyList_GET_SIZE(keys)) Py_RETURN_NONE;
            Py_ssize_t pos = 0, j = 0;
            PyObject *key, *value;
            while (PyDict_Next(state, &pos, &key, &value)) {
                if (key != PyList_GET_ITEM(keys, j) || value != PyList_GET_ITEM(values, j) || !PyDict_Check(value)) Py_RETURN_NONE;
                for (Py_ssize_t k = 0; k < PyTuple_GET_SIZE(names); k++, state_words += WORDS)
                    if (!same(PyDict_GetItem(value, PyTuple_GET_ITEM(names, k)), state_words)) Py_RETURN_NONE;
                j++;
            }
            PyObject* grads = PyList_New(n);
            if (grads == nullptr) return nullptr;
            *plain = 1;
            *written = 0;
            for (i = 0; i < n; i++) {
                const long long* w = words + (WORDS + 2) * i;
                const at::Tensor& g = THPVariable_Unpack(PyList_GET_ITEM(params, i)).grad();
                PyObject* o = THPVariable_Wrap(g);  // None for none
                if (o == nullptr) {
                    Py_DECREF(grads);
                    return nullptr;
                }
                PyList_SET_ITEM(grads, i, o);
                if ((o != Py_None) != (w[WORDS] != 0)) {
                    Py_DECREF(grads);
                    Py_RETURN_NONE;
                }
                long long d[WORDS];
                describe(o, d);
                at[i] = d[0];
                if (o != Py_None && w[2] > 0 && versions[i] != -1 &&
                    THPVariable_Unpack(PyList_GET_ITEM(params, i))._version() != versions[i])
                    *written = 1;
                if (o != Py_None && (d[1] != w[1] || d[2] != w[WORDS + 1] || d[3] != w[3] || !d[4])) *plain = 0;
            }
            return grads;
        },
        nullptr);
}

// out[places[i]]: the version of parameter i of a list, if it is one of 16 bits.  0, or -1
int gsr_tensors_versions(PyObject* params, const int* places, long long* out) {
    return guarded(
        [&] {
            for (Py_ssize_t i = 0; i < PyList_GET_SIZE(params); i++) {
                const at::Tensor& p = THPVariable_Unpack(PyList_GET_ITEM(params, i));
                if (p.scalar_type() != at::kFloat) out[places[i]] = p._version();
            }
            return 0;
        },
        -1);
}

}  // extern "C"
