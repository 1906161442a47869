// The host side of the calls in neoml_b200/ops.py that a network issues by the dozen, in native code: argument checks, the
// result and work-space tensors, and the C ABI call.  A layer's kernels take a few microseconds at small batches; the
// same steps in Python (two torch.empty, a ctypes structure or two, fifteen converted arguments) took 15-20 us a call,
// here 5-7.
//
// Every function takes positional arguments and returns the result tensor; an int is the C ABI's error code; None means
// that an argument is not what this path takes (not a plain contiguous fp32 CUDA tensor, a size that does not fit): the
// caller then runs its own code, which raises or handles it.  Nothing is kept between calls.
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/python_arg_parser.h>
#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include "../../include/neoml_b200.h"

#include <exception>

namespace {

struct NotHere {}; // "run the Python code"

const at::Tensor& tensor(PyObject* o)
{
	if(!THPVariable_CheckExact(o)) throw NotHere();
	const at::Tensor& t = THPVariable_Unpack(o);
	if(!t.has_storage() || !t.is_cuda() || !t.is_contiguous()) throw NotHere();
	return t;
}

const float* data(PyObject* o) // None: null
{
	return o == Py_None ? nullptr : static_cast<const float*>(tensor(o).data_ptr());
}

const at::Tensor& fp32(PyObject* o)
{
	const at::Tensor& t = tensor(o);
	if(t.scalar_type() != at::kFloat) throw NotHere();
	return t;
}

int integer(PyObject* o)
{
	if(!PyLong_Check(o)) throw NotHere();
	int overflow = 0;
	const long v = PyLong_AsLongAndOverflow(o, &overflow);
	if(overflow != 0 || v < INT32_MIN || v > INT32_MAX) throw NotHere();
	return static_cast<int>(v);
}

int size_of(const at::Tensor& t, int dim)
{
	const int64_t v = t.size(dim);
	if(v > INT32_MAX) throw NotHere();
	return static_cast<int>(v);
}

float number(PyObject* o)
{
	if(PyFloat_CheckExact(o)) return static_cast<float>(PyFloat_AS_DOUBLE(o));
	return static_cast<float>(integer(o));
}

bool truth(PyObject* o)
{
	const int v = PyObject_IsTrue(o);
	if(v < 0) { PyErr_Clear(); throw NotHere(); }
	return v != 0;
}

at::Tensor floats_like(const at::Tensor& like, at::IntArrayRef sizes)
{
	return at::empty(sizes, at::TensorOptions().dtype(at::kFloat).device(like.device()));
}

void* stream()
{
	return c10::cuda::getCurrentCUDAStream().stream();
}

template<typename F>
int without_gil(F&& f)
{
	int rc;
	Py_BEGIN_ALLOW_THREADS
	rc = f();
	Py_END_ALLOW_THREADS
	return rc;
}

PyObject* answer(int rc, const at::Tensor& result)
{
	return rc != NB200_OK ? PyLong_FromLong(rc) : THPVariable_Wrap(result);
}

template<typename F>
PyObject* guarded(Py_ssize_t n, Py_ssize_t expected, F&& f)
{
	if(n != expected) {
		PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", expected, n);
		return nullptr;
	}
	// a mode that wants to see torch.empty and the like sees them in the Python code
	if(at::impl::torch_function_mode_enabled()) Py_RETURN_NONE;
	try {
		return f();
	} catch(const NotHere&) {
		Py_RETURN_NONE;
	} catch(const c10::OutOfMemoryError&) {
		Py_RETURN_NONE; // the Python code does without the work space, or raises torch's own error
	} catch(const std::exception& e) {
		PyErr_SetString(PyExc_RuntimeError, e.what());
		return nullptr;
	}
}

nb200_epilogue epilogue(PyObject* bias, PyObject* residual, int ldResidual, PyObject* act, PyObject* actParam, bool accumulate)
{
	nb200_epilogue e = {};
	e.bias = data(bias);
	e.residual = data(residual);
	e.ld_residual = ldResidual;
	e.act = integer(act);
	e.act_param = number(actParam);
	e.accumulate = accumulate ? 1 : 0;
	return e;
}

int out_size(int size, int filter, int pad, int stride, int dilation)
{
	if(stride <= 0) throw NotHere();
	const int span = size - (filter - 1) * dilation - 1 + 2 * pad;
	if(span < 0) throw NotHere();
	return 1 + span / stride;
}

// source, filter, free_term, result, pad_h, pad_w, stride_h, stride_w, dil_h, dil_w, residual, act, act_param, precision, use_scratch
PyObject* blob_convolution(PyObject*, PyObject* const* a, Py_ssize_t count)
{
	return guarded(count, 15, [&]() -> PyObject* {
		const at::Tensor &x = fp32(a[0]), &f = fp32(a[1]);
		if(x.dim() != 4 || f.dim() != 4 || f.size(3) != x.size(3)) throw NotHere();
		nb200_conv_desc d = {};
		d.batch = size_of(x, 0); d.h = size_of(x, 1); d.w = size_of(x, 2); d.c = size_of(x, 3);
		d.k = size_of(f, 0); d.r = size_of(f, 1); d.s = size_of(f, 2);
		d.pad_h = integer(a[4]); d.pad_w = integer(a[5]); d.stride_h = integer(a[6]); d.stride_w = integer(a[7]);
		d.dil_h = integer(a[8]); d.dil_w = integer(a[9]);
		d.ho = out_size(d.h, d.r, d.pad_h, d.stride_h, d.dil_h);
		d.wo = out_size(d.w, d.s, d.pad_w, d.stride_w, d.dil_w);
		const nb200_epilogue e = epilogue(a[2], a[10], d.k, a[11], a[12], false);
		const int precision = integer(a[13]);
		at::Tensor y = a[3] == Py_None ? floats_like(x, { d.batch, d.ho, d.wo, d.k }) : tensor(a[3]);
		const size_t need = truth(a[14]) ? nb200_blob_convolution_scratch_floats(&d) : 0;
		at::Tensor scratch;
		if(need > 0) scratch = floats_like(x, { static_cast<int64_t>(need) });
		void* const s = stream();
		const float *xp = static_cast<const float*>(x.data_ptr()), *fp = static_cast<const float*>(f.data_ptr());
		float *yp = static_cast<float*>(y.data_ptr()), *sp = need > 0 ? static_cast<float*>(scratch.data_ptr()) : nullptr;
		return answer(without_gil([&] { return nb200_blob_convolution(s, &d, xp, fp, yp, sp, &e, precision); }), y);
	});
}

// first, second, result, m, k, n, lda, ldb, ldc, free_term, residual, act, act_param, accumulate, precision, use_scratch
PyObject* multiply_by_transposed(PyObject*, PyObject* const* a, Py_ssize_t count)
{
	return guarded(count, 16, [&]() -> PyObject* {
		const at::Tensor &first = fp32(a[0]), &second = fp32(a[1]);
		const int m = integer(a[3]), k = integer(a[4]), n = integer(a[5]), lda = integer(a[6]), ldb = integer(a[7]), ldc = integer(a[8]);
		if(m < 0 || ldc < 0) throw NotHere();
		const nb200_epilogue e = epilogue(a[9], a[10], ldc, a[11], a[12], truth(a[13]));
		const int precision = integer(a[14]);
		at::Tensor result = a[2] == Py_None ? floats_like(first, { m, ldc }) : tensor(a[2]);
		const size_t need = truth(a[15]) ? nb200_matrix_product_scratch_floats(1, m, n, k, ldb) : 0;
		at::Tensor scratch;
		if(need > 0) scratch = floats_like(first, { static_cast<int64_t>(need) });
		void* const s = stream();
		const float *ap = static_cast<const float*>(first.data_ptr()), *bp = static_cast<const float*>(second.data_ptr());
		float *cp = static_cast<float*>(result.data_ptr()), *sp = need > 0 ? static_cast<float*>(scratch.data_ptr()) : nullptr;
		return answer(without_gil([&] {
			return need > 0 ? nb200_multiply_matrix_by_transposed_matrix_with_scratch(s, 1, ap, m, k, lda, bp, n, ldb, cp, ldc, sp, &e, precision)
				: nb200_multiply_matrix_by_transposed_matrix(s, ap, m, k, lda, bp, n, ldb, cp, ldc, &e, precision);
		}), result);
	});
}

int batch_product(void* s, int batch, const float* a, int m, int k, const float* b, int n, float* c, float* scratch, int precision)
{
	return scratch != nullptr
		? nb200_multiply_matrix_by_transposed_matrix_with_scratch(s, batch, a, m, k, k, b, n, k, c, n, scratch, nullptr, precision)
		: nb200_batch_multiply_matrix_by_transposed_matrix(s, batch, a, m, k, b, n, c, nullptr, precision);
}

// first [b, m, k], second [b, n, k], result, precision, use_scratch
PyObject* batch_multiply_by_transposed(PyObject*, PyObject* const* a, Py_ssize_t count)
{
	return guarded(count, 5, [&]() -> PyObject* {
		const at::Tensor &first = fp32(a[0]), &second = fp32(a[1]);
		if(first.dim() != 3 || second.dim() != 3) throw NotHere();
		const int b = size_of(first, 0), m = size_of(first, 1), k = size_of(first, 2), n = size_of(second, 1);
		const int precision = integer(a[3]);
		at::Tensor result = a[2] == Py_None ? floats_like(first, { b, m, n }) : tensor(a[2]);
		const size_t need = truth(a[4]) ? nb200_matrix_product_scratch_floats(b, m, n, k, k) : 0;
		at::Tensor scratch;
		if(need > 0) scratch = floats_like(first, { static_cast<int64_t>(need) });
		void* const s = stream();
		const float *ap = static_cast<const float*>(first.data_ptr()), *bp = static_cast<const float*>(second.data_ptr());
		float *cp = static_cast<float*>(result.data_ptr()), *sp = need > 0 ? static_cast<float*>(scratch.data_ptr()) : nullptr;
		return answer(without_gil([&] { return batch_product(s, b, ap, m, k, bp, n, cp, sp, precision); }), result);
	});
}

// first [b, m, k], second [b, k, n], result, precision: with work space, k and n at least four (the second operand is
// transposed once)
PyObject* multiply_by_matrix(PyObject*, PyObject* const* a, Py_ssize_t count)
{
	return guarded(count, 4, [&]() -> PyObject* {
		const at::Tensor &first = fp32(a[0]), &second = fp32(a[1]);
		if(first.dim() != 3 || second.dim() != 3) throw NotHere();
		const int b = size_of(first, 0), m = size_of(first, 1), k = size_of(first, 2), n = size_of(second, 2);
		if(k < 4 || n < 4) throw NotHere();
		const int precision = integer(a[3]);
		at::Tensor result = a[2] == Py_None ? floats_like(first, { b, m, n }) : tensor(a[2]);
		const size_t need = nb200_matrix_product_scratch_floats(b, m, n, k, k);
		const int64_t across = (static_cast<int64_t>(b) * n * k + 3) / 4 * 4;
		// one block: the transposed operand, then the product's own room
		at::Tensor room = floats_like(first, { across + static_cast<int64_t>(need) });
		void* const s = stream();
		const float *ap = static_cast<const float*>(first.data_ptr()), *bp = static_cast<const float*>(second.data_ptr());
		float *cp = static_cast<float*>(result.data_ptr()), *tp = static_cast<float*>(room.data_ptr());
		return answer(without_gil([&] {
			const int rc = nb200_transpose_matrix(s, b, bp, k, 1, n, 1, tp);
			return rc != NB200_OK ? rc : batch_product(s, b, ap, m, k, tp, n, cp, need > 0 ? tp + across : nullptr, precision);
		}), result);
	});
}

// batch, first, height, medium, width, channels, result
PyObject* transpose(PyObject*, PyObject* const* a, Py_ssize_t count)
{
	return guarded(count, 7, [&]() -> PyObject* {
		const int batch = integer(a[0]), h = integer(a[2]), m = integer(a[3]), w = integer(a[4]), c = integer(a[5]);
		const at::Tensor& first = fp32(a[1]);
		at::Tensor result = a[6] == Py_None ? floats_like(first, first.sizes()) : tensor(a[6]);
		void* const s = stream();
		const float* ap = static_cast<const float*>(first.data_ptr());
		float* rp = static_cast<float*>(result.data_ptr());
		return answer(without_gil([&] { return nb200_transpose_matrix(s, batch, ap, h, m, w, c, rp); }), result);
	});
}

// op code, first, second, scalar, value, result, count (None: the result's size); first or result given
PyObject* vector_op(PyObject*, PyObject* const* a, Py_ssize_t count)
{
	return guarded(count, 7, [&]() -> PyObject* {
		const int op = integer(a[0]);
		const float *first = data(a[1]), *second = data(a[2]), *scalar = data(a[3]);
		const float value = number(a[4]);
		if(a[5] == Py_None && a[1] == Py_None) throw NotHere();
		at::Tensor result = a[5] == Py_None ? floats_like(fp32(a[1]), tensor(a[1]).sizes()) : tensor(a[5]);
		const int64_t n = a[6] == Py_None ? result.numel() : integer(a[6]);
		if(n > INT32_MAX) throw NotHere();
		void* const s = stream();
		float* rp = static_cast<float*>(result.data_ptr());
		return answer(without_gil([&] { return nb200_vector_op(s, op, first, second, scalar, value, rp, static_cast<int>(n)); }), result);
	});
}

// ---- operators of language models: fp32, fp16 and bf16 data on the device that it is on ------------------------------

PyObject* g_parameter = nullptr; // torch.nn.Parameter, held for as long as the process lives

const at::Tensor& any_tensor(PyObject* o) // parameters too
{
	if(!THPVariable_CheckExact(o) && reinterpret_cast<PyObject*>(Py_TYPE(o)) != g_parameter) throw NotHere();
	const at::Tensor& t = THPVariable_Unpack(o);
	if(!t.has_storage() || !t.is_cuda() || t.is_conj() || t.is_neg()) throw NotHere();
	return t;
}

int type_code(const at::Tensor& t)
{
	switch(t.scalar_type()) {
		case at::kFloat: return NB200_TYPE_FP32;
		case at::kHalf: return NB200_TYPE_FP16;
		case at::kBFloat16: return NB200_TYPE_BF16;
		default: throw NotHere();
	}
}

struct Matrix {
	int height, width;
	long long row;
};
Matrix matrix(const at::Tensor& t)
{
	const int64_t dims = t.dim();
	if(dims < 1 || t.size(dims - 1) < 1) throw NotHere();
	Matrix m;
	m.width = size_of(t, static_cast<int>(dims) - 1);
	m.row = m.width;
	if(dims == 2 && t.size(0) > 1) {
		if((m.width > 1 && t.stride(1) != 1) || t.stride(0) < m.width) throw NotHere();
		m.height = size_of(t, 0);
		m.row = t.stride(0);
		return m;
	}
	if(!t.is_contiguous()) throw NotHere();
	const int64_t rows = t.numel() / m.width;
	if(rows > INT32_MAX) throw NotHere();
	m.height = static_cast<int>(rows);
	return m;
}

// An optional contiguous vector of `count` elements of the type, on the device.
void* vector(PyObject* o, int64_t count, at::ScalarType type, const at::Device& device)
{
	if(o == Py_None) return nullptr;
	const at::Tensor& t = any_tensor(o);
	if(t.numel() != count || !t.is_contiguous() || t.scalar_type() != type || t.device() != device) throw NotHere();
	return t.data_ptr();
}
template<typename T>
T* vector_of(PyObject* o, int64_t count, at::ScalarType type, const at::Device& device)
{
	return static_cast<T*>(vector(o, count, type, device));
}

at::Tensor empty(at::IntArrayRef sizes, at::ScalarType type, const at::Device& device)
{
	return at::empty(sizes, at::TensorOptions().dtype(type).device(device));
}
at::Tensor empty_or(PyObject* given, const at::Tensor& like) // None: a new dense tensor
{
	if(given == Py_None) return empty(like.sizes(), like.scalar_type(), like.device());
	const at::Tensor& t = any_tensor(given);
	if(t.sizes() != like.sizes() || t.scalar_type() != like.scalar_type() || t.device() != like.device()) throw NotHere();
	return t;
}

// The device of the call: current while it lasts, with torch's current stream of that device.
struct On {
	c10::cuda::OptionalCUDAGuard guard;
	void* stream;
	explicit On(const at::Device& device)
	{
		if(c10::cuda::current_device() != device.index()) guard.set_device(device);
		stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
	}
};

PyObject* answers(int rc, std::initializer_list<const at::Tensor*> results) // null: None
{
	if(rc != NB200_OK) return PyLong_FromLong(rc);
	PyObject* tuple = PyTuple_New(static_cast<Py_ssize_t>(results.size()));
	if(tuple == nullptr) return nullptr;
	Py_ssize_t i = 0;
	for(const at::Tensor* t : results) {
		PyObject* o = t == nullptr ? Py_NewRef(Py_None) : THPVariable_Wrap(*t);
		if(o == nullptr) {
			Py_DECREF(tuple);
			return nullptr;
		}
		PyTuple_SET_ITEM(tuple, i++, o);
	}
	return tuple;
}

at::ScalarType parameter_type(std::initializer_list<PyObject*> parameters, const at::Tensor& x)
{
	for(PyObject* o : parameters) {
		if(o == Py_None) continue;
		const at::ScalarType type = any_tensor(o).scalar_type();
		if(type != x.scalar_type() && type != at::kFloat) throw NotHere();
		return type;
	}
	return x.scalar_type();
}
int code_of(at::ScalarType type)
{
	return type == at::kFloat ? NB200_TYPE_FP32 : type == at::kHalf ? NB200_TYPE_FP16 : NB200_TYPE_BF16;
}

// source, scale, free_term, epsilon, result
PyObject* layer_normalization(PyObject*, PyObject* const* a, Py_ssize_t count)
{
	return guarded(count, 5, [&]() -> PyObject* {
		const at::Tensor& x = any_tensor(a[0]);
		const int type = type_code(x);
		const Matrix m = matrix(x);
		const at::Device device = x.device();
		const at::ScalarType parameter = parameter_type({ a[1], a[2] }, x);
		const void *scale = vector(a[1], m.width, parameter, device), *free = vector(a[2], m.width, parameter, device);
		const float epsilon = number(a[3]);
		at::Tensor y = empty_or(a[4], x);
		const Matrix my = matrix(y);
		const at::IntArrayRef rows = x.sizes().slice(0, x.dim() - 1);
		at::Tensor mean = empty(rows, at::kFloat, device), inverse = empty(rows, at::kFloat, device);
		const On on(device);
		const void* xp = x.data_ptr();
		void* yp = y.data_ptr();
		float *mp = static_cast<float*>(mean.data_ptr()), *ip = static_cast<float*>(inverse.data_ptr());
		const int rc = without_gil([&] {
			return nb200_layer_normalization(on.stream, type, code_of(parameter), xp, m.height, m.width, m.row, scale, free, epsilon, yp, my.row, mp, ip);
		});
		return answers(rc, { &y, &mean, &inverse });
	});
}

// result_diff, source, mean, inverse_deviation, scale (not None, or parameters False), source_diff, parameters
PyObject* layer_normalization_backward(PyObject*, PyObject* const* a, Py_ssize_t count)
{
	return guarded(count, 7, [&]() -> PyObject* {
		const at::Tensor &dy = any_tensor(a[0]), &x = any_tensor(a[1]);
		const int type = type_code(x);
		if(dy.sizes() != x.sizes() || dy.scalar_type() != x.scalar_type() || dy.device() != x.device()) throw NotHere();
		const Matrix m = matrix(x), md = matrix(dy);
		const at::Device device = x.device();
		const bool parameters = truth(a[6]);
		if(parameters && a[4] == Py_None) throw NotHere();
		const at::ScalarType parameter = parameter_type({ a[4] }, x);
		const float *mean = vector_of<float>(a[2], m.height, at::kFloat, device), *inverse = vector_of<float>(a[3], m.height, at::kFloat, device);
		if(mean == nullptr || inverse == nullptr) throw NotHere();
		const void* scale = vector(a[4], m.width, parameter, device);
		at::Tensor dx = empty_or(a[5], x);
		const Matrix mx = matrix(dx);
		const On on(device);
		at::Tensor ds, db, scratch;
		void *dsp = nullptr, *dbp = nullptr;
		float* room = nullptr;
		if(parameters) {
			ds = empty({ m.width }, parameter, device);
			db = empty({ m.width }, parameter, device);
			scratch = empty({ static_cast<int64_t>(nb200_layer_normalization_backward_scratch_floats(type, m.height, m.width)) }, at::kFloat, device);
			dsp = ds.data_ptr();
			dbp = db.data_ptr();
			room = static_cast<float*>(scratch.data_ptr());
		}
		const void *xp = x.data_ptr(), *dyp = dy.data_ptr();
		void* dxp = dx.data_ptr();
		const int rc = without_gil([&] {
			return nb200_layer_normalization_backward(on.stream, type, code_of(parameter), dyp, md.row, xp, m.height, m.width, m.row, scale, mean,
				inverse, dxp, mx.row, dsp, dbp, room);
		});
		return answers(rc, { &dx, parameters ? &ds : nullptr, parameters ? &db : nullptr });
	});
}

struct Sequences {
	nb200_recurrence_desc desc;
	const at::Tensor* z;
	const void *zp, *fp, *ip;
};
void steps(const at::Tensor& t, const at::Tensor& like, long long* batch, long long* row)
{
	if(t.sizes() != like.sizes() || t.scalar_type() != like.scalar_type() || t.device() != like.device()
		|| (t.size(2) > 1 && t.stride(2) != 1)) throw NotHere();
	*batch = t.size(0) > 1 ? t.stride(0) : 0;
	*row = t.size(1) > 1 ? t.stride(1) : 0;
}
Sequences sequences(PyObject* update, PyObject* forget, PyObject* input)
{
	Sequences s = {};
	const at::Tensor &z = any_tensor(update), &f = any_tensor(forget);
	if(z.dim() != 3) throw NotHere();
	s.z = &z;
	s.desc.batch = size_of(z, 0); s.desc.length = size_of(z, 1); s.desc.channels = size_of(z, 2);
	steps(z, z, &s.desc.update_batch, &s.desc.update_row);
	steps(f, z, &s.desc.forget_batch, &s.desc.forget_row);
	s.zp = z.data_ptr();
	s.fp = f.data_ptr();
	if(input != Py_None) {
		const at::Tensor& i = any_tensor(input);
		steps(i, z, &s.desc.input_batch, &s.desc.input_row);
		s.ip = i.data_ptr();
		if(s.ip == nullptr) throw NotHere(); // an empty one: the Python code tells it from none
	}
	return s;
}

// update, forget, input, initial_state, lengths, result, final_state
PyObject* gated_recurrence(PyObject*, PyObject* const* a, Py_ssize_t count)
{
	return guarded(count, 7, [&]() -> PyObject* {
		const Sequences s = sequences(a[0], a[1], a[2]);
		const at::Tensor& z = *s.z;
		const int type = type_code(z);
		const at::Device device = z.device();
		const int64_t states = z.size(0) * z.size(2);
		const float* first = vector_of<float>(a[3], states, at::kFloat, device);
		const int* lengths = vector_of<int>(a[4], z.size(0), at::kInt, device);
		at::Tensor h = empty_or(a[5], z);
		if(!h.is_contiguous()) throw NotHere();
		float* last = vector_of<float>(a[6], states, at::kFloat, device);
		at::Tensor state = a[6] == Py_None ? empty({ z.size(0), z.size(2) }, at::kFloat, device) : any_tensor(a[6]);
		if(a[6] == Py_None) last = static_cast<float*>(state.data_ptr());
		const On on(device);
		void* hp = h.data_ptr();
		const int rc = without_gil([&] { return nb200_gated_recurrence(on.stream, type, &s.desc, s.zp, s.fp, s.ip, first, lengths, hp, last); });
		return answers(rc, { &h, &state });
	});
}

// result_diff, result, update, forget, input, initial_state, final_state_diff, lengths
PyObject* gated_recurrence_backward(PyObject*, PyObject* const* a, Py_ssize_t count)
{
	return guarded(count, 8, [&]() -> PyObject* {
		const Sequences s = sequences(a[2], a[3], a[4]);
		const at::Tensor &z = *s.z, &dh = any_tensor(a[0]), &h = any_tensor(a[1]);
		const int type = type_code(z);
		const at::Device device = z.device();
		long long dhBatch, dhRow, hBatch, hRow;
		steps(dh, z, &dhBatch, &dhRow);
		steps(h, z, &hBatch, &hRow);
		if(!h.is_contiguous()) throw NotHere();
		const int64_t states = z.size(0) * z.size(2);
		const float *first = vector_of<float>(a[5], states, at::kFloat, device), *lastDiff = vector_of<float>(a[6], states, at::kFloat, device);
		const int* lengths = vector_of<int>(a[7], z.size(0), at::kInt, device);
		const bool input = a[4] != Py_None;
		at::Tensor dz = empty(z.sizes(), z.scalar_type(), device), df = empty(z.sizes(), z.scalar_type(), device), di;
		if(input) di = empty(z.sizes(), z.scalar_type(), device);
		at::Tensor dfirst = empty({ z.size(0), z.size(2) }, at::kFloat, device);
		const On on(device);
		const void *dhp = dh.data_ptr(), *hp = h.data_ptr();
		void *dzp = dz.data_ptr(), *dfp = df.data_ptr(), *dip = input ? di.data_ptr() : nullptr;
		float* dfirstp = static_cast<float*>(dfirst.data_ptr());
		const int rc = without_gil([&] {
			return nb200_gated_recurrence_backward(on.stream, type, &s.desc, dhp, dhBatch, dhRow, hp, s.zp, s.fp, s.ip, first, lastDiff, lengths, dzp, dfp,
				dip, dfirstp);
		});
		return answers(rc, { &dz, &df, input ? &di : nullptr, &dfirst });
	});
}

struct Taught {
	const at::Tensor* logits;
	Matrix m;
	int type, teacherType, kept;
	const void* teacher;
	const int* indices;
	float temperature;
};
Taught taught(PyObject* logits, PyObject* teacher, PyObject* indices, PyObject* temperature)
{
	Taught t = {};
	const at::Tensor &x = any_tensor(logits), &top = any_tensor(teacher), &at = any_tensor(indices);
	t.logits = &x;
	t.type = type_code(x);
	t.m = matrix(x);
	if(top.dim() != x.dim() || top.sizes() != at.sizes() || top.sizes().slice(0, top.dim() - 1) != x.sizes().slice(0, x.dim() - 1)) throw NotHere();
	t.kept = size_of(top, static_cast<int>(top.dim()) - 1);
	const at::ScalarType type = parameter_type({ teacher }, x);
	t.teacherType = code_of(type);
	t.teacher = vector(teacher, static_cast<int64_t>(t.m.height) * t.kept, type, x.device());
	t.indices = vector_of<int>(indices, static_cast<int64_t>(t.m.height) * t.kept, at::kInt, x.device());
	if(!PyFloat_CheckExact(temperature)) throw NotHere();
	const double tau = PyFloat_AS_DOUBLE(temperature);
	if(!(tau > 0.0) || !(tau < 1e38)) throw NotHere();
	t.temperature = static_cast<float>(tau);
	return t;
}

// logits, teacher_logits, teacher_indices, temperature
PyObject* distillation_loss(PyObject*, PyObject* const* a, Py_ssize_t count)
{
	return guarded(count, 4, [&]() -> PyObject* {
		const Taught t = taught(a[0], a[1], a[2], a[3]);
		const at::Tensor& x = *t.logits;
		const at::IntArrayRef rows = x.sizes().slice(0, x.dim() - 1);
		at::Tensor loss = empty(rows, at::kFloat, x.device()), logSum = empty(rows, at::kFloat, x.device());
		const On on(x.device());
		const void* xp = x.data_ptr();
		float *lp = static_cast<float*>(loss.data_ptr()), *sp = static_cast<float*>(logSum.data_ptr());
		const int rc = without_gil([&] {
			return nb200_distillation_loss(on.stream, t.type, t.teacherType, xp, t.m.height, t.m.width, t.m.row, t.teacher, t.indices, t.kept,
				t.temperature, lp, sp);
		});
		return answers(rc, { &loss, &logSum });
	});
}

// loss_diff, logits, teacher_logits, teacher_indices, log_sum, temperature, result
PyObject* distillation_loss_backward(PyObject*, PyObject* const* a, Py_ssize_t count)
{
	return guarded(count, 7, [&]() -> PyObject* {
		const Taught t = taught(a[1], a[2], a[3], a[5]);
		const at::Tensor& x = *t.logits;
		const float *diff = vector_of<float>(a[0], t.m.height, at::kFloat, x.device()), *logSum = vector_of<float>(a[4], t.m.height, at::kFloat, x.device());
		if(a[0] == Py_None || a[4] == Py_None) throw NotHere();
		at::Tensor out = empty_or(a[6], x);
		const Matrix mo = matrix(out);
		const On on(x.device());
		const void* xp = x.data_ptr();
		void* op = out.data_ptr();
		const int rc = without_gil([&] {
			return nb200_distillation_loss_backward(on.stream, t.type, t.teacherType, diff, xp, t.m.height, t.m.width, t.m.row, t.teacher, t.indices,
				t.kept, t.temperature, logSum, op, mo.row);
		});
		return answer(rc, out);
	});
}

struct Head {
	const at::Tensor *x, *w;
	Matrix m, mw;
	int type;
	const int* labels;
};
Head head(PyObject* hidden, PyObject* weights, PyObject* labels)
{
	Head h = {};
	const at::Tensor &x = any_tensor(hidden), &w = any_tensor(weights);
	h.x = &x;
	h.w = &w;
	h.type = type_code(x);
	h.m = matrix(x);
	if(w.dim() != 2 || w.size(0) < 1 || w.scalar_type() != x.scalar_type() || w.device() != x.device()) throw NotHere();
	h.mw = matrix(w);
	if(h.mw.width != h.m.width || any_tensor(labels).sizes() != x.sizes().slice(0, x.dim() - 1)) throw NotHere();
	h.labels = vector_of<int>(labels, h.m.height, at::kInt, x.device());
	return h;
}
at::Tensor head_scratch(const Head& h, bool backward)
{
	const size_t need = nb200_vocabulary_cross_entropy_scratch_bytes(h.type, h.x->data_ptr(), h.m.height, h.m.width, h.m.row, h.w->data_ptr(),
		h.mw.height, h.mw.row, backward ? 1 : 0);
	return empty({ static_cast<int64_t>(need) }, at::kByte, h.x->device());
}

// hidden, weights, labels
PyObject* vocabulary_cross_entropy(PyObject*, PyObject* const* a, Py_ssize_t count)
{
	return guarded(count, 3, [&]() -> PyObject* {
		const Head h = head(a[0], a[1], a[2]);
		const at::Device device = h.x->device();
		const at::IntArrayRef rows = h.x->sizes().slice(0, h.x->dim() - 1);
		at::Tensor loss = empty(rows, at::kFloat, device), logSum = empty(rows, at::kFloat, device);
		const On on(device);
		at::Tensor scratch = head_scratch(h, false);
		const void *xp = h.x->data_ptr(), *wp = h.w->data_ptr();
		float *lp = static_cast<float*>(loss.data_ptr()), *sp = static_cast<float*>(logSum.data_ptr());
		void* room = scratch.data_ptr();
		const int rc = without_gil([&] {
			return nb200_vocabulary_cross_entropy(on.stream, h.type, xp, h.m.height, h.m.width, h.m.row, wp, h.mw.height, h.mw.row, h.labels, lp, sp, room);
		});
		return answers(rc, { &loss, &logSum });
	});
}

// loss_diff, hidden, weights, labels, log_sum, hidden_diff, weights_diff (True, a tensor, or False or None: not wanted)
PyObject* vocabulary_cross_entropy_backward(PyObject*, PyObject* const* a, Py_ssize_t count)
{
	return guarded(count, 7, [&]() -> PyObject* {
		const Head h = head(a[1], a[2], a[3]);
		const at::Device device = h.x->device();
		if(a[0] == Py_None || a[4] == Py_None) throw NotHere();
		const float *diff = vector_of<float>(a[0], h.m.height, at::kFloat, device), *logSum = vector_of<float>(a[4], h.m.height, at::kFloat, device);
		at::Tensor dx, dw;
		void *dxp = nullptr, *dwp = nullptr;
		long long dxRow = 0, dwRow = 0;
		const bool wantsX = a[5] != Py_False && a[5] != Py_None, wantsW = a[6] != Py_False && a[6] != Py_None;
		if(wantsX) {
			dx = empty_or(a[5] == Py_True ? Py_None : a[5], *h.x);
			dxp = dx.data_ptr();
			dxRow = matrix(dx).row;
		}
		if(wantsW) {
			dw = empty_or(a[6] == Py_True ? Py_None : a[6], *h.w);
			dwp = dw.data_ptr();
			dwRow = matrix(dw).row;
		}
		const On on(device);
		at::Tensor scratch = head_scratch(h, true);
		const void *xp = h.x->data_ptr(), *wp = h.w->data_ptr();
		void* room = scratch.data_ptr();
		const int rc = without_gil([&] {
			return nb200_vocabulary_cross_entropy_backward(on.stream, h.type, diff, xp, h.m.height, h.m.width, h.m.row, wp, h.mw.height, h.mw.row,
				h.labels, logSum, dxp, dxRow, dwp, dwRow, room);
		});
		return answers(rc, { wantsX ? &dx : nullptr, wantsW ? &dw : nullptr });
	});
}

PyMethodDef methods[] = {
#define FAST(name) { #name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr }
	FAST(blob_convolution), FAST(multiply_by_transposed), FAST(batch_multiply_by_transposed), FAST(multiply_by_matrix),
	FAST(transpose), FAST(vector_op), FAST(layer_normalization), FAST(layer_normalization_backward), FAST(gated_recurrence),
	FAST(gated_recurrence_backward), FAST(distillation_loss), FAST(distillation_loss_backward), FAST(vocabulary_cross_entropy),
	FAST(vocabulary_cross_entropy_backward),
#undef FAST
	{ nullptr, nullptr, 0, nullptr }
};

PyModuleDef module = { PyModuleDef_HEAD_INIT, "_ops_native", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr };

} // namespace

PyMODINIT_FUNC PyInit__ops_native()
{
	PyObject* const nn = PyImport_ImportModule("torch.nn.parameter");
	if(nn == nullptr) return nullptr;
	g_parameter = PyObject_GetAttrString(nn, "Parameter");
	Py_DECREF(nn);
	if(g_parameter == nullptr) return nullptr;
	return PyModule_Create(&module);
}
