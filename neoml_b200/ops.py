"""Host-side mirror of the IMathEngine methods on the inference hot path, over torch CUDA tensors.

torch is used for device memory and streams only; every computation is a call into the C ABI
(include/neoml_b200.h) on the tensors' device pointers, enqueued on torch's current stream.
Method names and argument meaning follow NeoMathEngine/include/NeoMathEngine/NeoMathEngine.h; blobs are
channels-last ``[batch, height, width, channels]`` fp32 tensors, filters ``[count, height, width, channels]``.

The operators of language models at the end of the file (normalisation, recurrence, losses) take fp32, fp16 or bf16 data
and run on the device that their tensors are on, on torch's current stream of that device.  What they record nowhere is a
gradient: the backward pass of each is a call of its own, as in NeoML's engine.
"""
from __future__ import annotations

import ctypes as C
import importlib.machinery
import importlib.util
import warnings

import torch

from . import _capi as capi
from ._capi import (ACT_HSWISH, ACT_NONE, ACT_RELU, PREC_3XTF32, PREC_FP32_SIMT, PREC_TF32, VEC)  # noqa: F401


_native_module = None


class _DeclinesAll:
    """In the place of a native half that has not been built for this interpreter and torch."""
    def __getattr__(self, name):
        return lambda *args: None


def _native():
    """The native half of the calls below (bindings/ops_native.cpp): it answers None for arguments that it does not take,
    and the Python code after the call then raises or handles them.  Its file is named after the torch and the interpreter
    that it was compiled for; without it the Python code makes every call, with the same kernels and more host time."""
    global _native_module
    if _native_module is None:
        capi.load()
        path = capi.native_path()
        if path.exists():
            loader = importlib.machinery.ExtensionFileLoader("_ops_native", str(path))
            module = importlib.util.module_from_spec(importlib.util.spec_from_loader("_ops_native", loader))
            loader.exec_module(module)
            _native_module = module
        else:
            warnings.warn(f"{path} is missing: calls take 10 us longer (python -m neoml_b200.build makes it)")
            _native_module = _DeclinesAll()
    return _native_module


def _checked(name: str, answer):
    if type(answer) is int:
        capi.check(name, answer)
    return answer


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _ptr(t: torch.Tensor | None) -> int | None:
    if t is None:
        return None
    assert t.is_cuda and t.is_contiguous(), "device-resident contiguous tensors only"
    return t.data_ptr()


def _f32(t: torch.Tensor) -> torch.Tensor:
    assert t.dtype == torch.float32
    return t


def _product_scratch(need: int, device) -> torch.Tensor | None:
    """Work space of a matrix product, or None where there is no room for it: the product then runs without, more slowly."""
    if not need:
        return None
    try:
        return torch.empty(need, dtype=torch.float32, device=device)
    except torch.cuda.OutOfMemoryError:
        return None


def _epilogue(bias=None, residual=None, ld_residual=0, act=ACT_NONE, act_param=0.0, accumulate=False,
              act_param_device=None):
    return capi.Epilogue(_ptr(bias), _ptr(residual), ld_residual, act, float(act_param), int(accumulate),
                         _ptr(act_param_device))


def conv_output_size(size: int, filt: int, pad: int, stride: int, dil: int = 1) -> int:
    """Output size rule of the reference (CpuMathEngineDnnConv.cpp:59-62)."""
    return 1 + (size - (filt - 1) * dil - 1 + 2 * pad) // stride


def MultiplyMatrixByTransposedMatrix(first, second, result=None, *, first_row_size=None, second_row_size=None,
                                     result_row_size=None, first_height=None, first_width=None, second_height=None,
                                     free_term=None, residual=None, act=ACT_NONE, act_param=0.0, accumulate=False,
                                     precision=PREC_3XTF32, use_scratch=True):
    """result[M x N] = first[M x K] * second[N x K]^T (+ fused tail).  2-D tensors give the shapes; pass explicit
    heights/widths/row sizes to address a sub-matrix of a larger buffer, as the reference allows.  With use_scratch
    (what the engine does with its stack allocator) the library gets work space for a prepared second operand and
    for split-K partial results."""
    m = first_height if first_height is not None else first.shape[0]
    k = first_width if first_width is not None else first.shape[1]
    n = second_height if second_height is not None else second.shape[0]
    lda = first_row_size if first_row_size is not None else k
    ldb = second_row_size if second_row_size is not None else k
    ldc = result_row_size if result_row_size is not None else n
    done = _native().multiply_by_transposed(first, second, result, m, k, n, lda, ldb, ldc, free_term, residual, act, act_param,
                                            accumulate, precision, use_scratch)
    if done is not None:
        return _checked("MultiplyMatrixByTransposedMatrix", done)
    if result is None:
        result = torch.empty((m, ldc), dtype=torch.float32, device=first.device)
    epi = _epilogue(free_term, residual, ldc, act, act_param, accumulate)
    lib = capi.load()
    scratch = _product_scratch(lib.nb200_matrix_product_scratch_floats(1, m, n, k, ldb) if use_scratch else 0, first.device)
    if scratch is not None:
        capi.check("MultiplyMatrixByTransposedMatrix", lib.nb200_multiply_matrix_by_transposed_matrix_with_scratch(
            _stream(), 1, _ptr(_f32(first)), m, k, lda, _ptr(_f32(second)), n, ldb, _ptr(result), ldc, _ptr(scratch),
            C.byref(epi), precision))
    else:
        capi.check("MultiplyMatrixByTransposedMatrix", lib.nb200_multiply_matrix_by_transposed_matrix(
            _stream(), _ptr(_f32(first)), m, k, lda, _ptr(_f32(second)), n, ldb, _ptr(result), ldc, C.byref(epi), precision))
    return result


def BatchMultiplyMatrixByTransposedMatrix(first, second, result=None, *, precision=PREC_3XTF32, use_scratch=True):
    """first [B, M, K], second [B, N, K] -> result [B, M, N]."""
    done = _native().batch_multiply_by_transposed(first, second, result, precision, use_scratch)
    if done is not None:
        return _checked("BatchMultiplyMatrixByTransposedMatrix", done)
    b, m, k = first.shape
    n = second.shape[1]
    if result is None:
        result = torch.empty((b, m, n), dtype=torch.float32, device=first.device)
    _batch_mmt(b, _f32(first), m, k, _f32(second), n, result, precision, use_scratch)
    return result


def _batch_mmt(b, first, m, k, second, n, result, precision, use_scratch):
    lib = capi.load()
    scratch = _product_scratch(lib.nb200_matrix_product_scratch_floats(b, m, n, k, k) if use_scratch else 0, first.device)
    if scratch is not None:
        capi.check("BatchMultiplyMatrixByTransposedMatrix", lib.nb200_multiply_matrix_by_transposed_matrix_with_scratch(
            _stream(), b, _ptr(first), m, k, k, _ptr(second), n, k, _ptr(result), n, _ptr(scratch), None, precision))
    else:
        capi.check("BatchMultiplyMatrixByTransposedMatrix", lib.nb200_batch_multiply_matrix_by_transposed_matrix(
            _stream(), b, _ptr(first), m, k, _ptr(second), n, _ptr(result), None, precision))


def MultiplyMatrixByMatrix(first, second, result=None, *, precision=PREC_3XTF32, use_scratch=True):
    """first [B, M, K] (or [M, K]), second [B, K, N] (or [K, N]) -> result [B, M, N].
    With use_scratch (what the engine does with its stack allocator) the second operand is transposed once into
    scratch and the product runs as A * (B^T)^T on the TMA-fed path; without, the kernel gathers the column-major
    operand itself."""
    squeeze = first.dim() == 2
    if squeeze:
        first, second = first.unsqueeze(0), second.unsqueeze(0)
    done = _native().multiply_by_matrix(first, second, result, precision) if use_scratch else None
    if done is not None:
        done = _checked("MultiplyMatrixByMatrix", done)
        return done[0] if squeeze else done
    b, m, k = first.shape
    n = second.shape[2]
    if result is None:
        result = torch.empty((b, m, n), dtype=torch.float32, device=first.device)
    lib = capi.load()
    if use_scratch and k >= 4 and n >= 4:
        transposed = torch.empty((b, n, k), dtype=torch.float32, device=first.device)
        capi.check("TransposeMatrix", lib.nb200_transpose_matrix(_stream(), b, _ptr(_f32(second)), k, 1, n, 1,
                                                                 _ptr(transposed)))
        _batch_mmt(b, _f32(first), m, k, transposed, n, result, precision, True)
    else:
        capi.check("MultiplyMatrixByMatrix", lib.nb200_multiply_matrix_by_matrix(
            _stream(), b, _ptr(_f32(first)), m, k, _ptr(_f32(second)), n, _ptr(result), None, precision))
    return result[0] if squeeze else result


def BlobConvolution(source, filter, free_term=None, result=None, *, padding=(0, 0), stride=(1, 1), dilation=(1, 1),
                    residual=None, act=ACT_NONE, act_param=0.0, precision=PREC_3XTF32, use_scratch=True):
    done = _native().blob_convolution(source, filter, free_term, result, padding[0], padding[1], stride[0], stride[1],
                                      dilation[0], dilation[1], residual, act, act_param, precision, use_scratch)
    if done is not None:
        return _checked("BlobConvolution", done)
    n, h, w, c = source.shape
    k, r, s, c2 = filter.shape
    assert c == c2
    ho = conv_output_size(h, r, padding[0], stride[0], dilation[0])
    wo = conv_output_size(w, s, padding[1], stride[1], dilation[1])
    if result is None:
        result = torch.empty((n, ho, wo, k), dtype=torch.float32, device=source.device)
    desc = capi.ConvDesc(n, h, w, c, k, r, s, padding[0], padding[1], stride[0], stride[1], dilation[0], dilation[1],
                         ho, wo)
    epi = _epilogue(free_term, residual, k, act, act_param)
    lib = capi.load()
    need = lib.nb200_blob_convolution_scratch_floats(C.byref(desc)) if use_scratch else 0
    scratch = torch.empty(need, dtype=torch.float32, device=source.device) if need else None
    capi.check("BlobConvolution", lib.nb200_blob_convolution(
        _stream(), C.byref(desc), _ptr(_f32(source)), _ptr(_f32(filter)), _ptr(result), _ptr(scratch), C.byref(epi),
        precision))
    return result


def BlobChannelwiseConvolution(source, filter, free_term=None, result=None, *, padding=(0, 0), stride=(1, 1),
                               act=ACT_NONE, act_param=0.0):
    n, h, w, c = source.shape
    r, s, c2 = filter.shape
    assert c == c2
    ho = conv_output_size(h, r, padding[0], stride[0])
    wo = conv_output_size(w, s, padding[1], stride[1])
    if result is None:
        result = torch.empty((n, ho, wo, c), dtype=torch.float32, device=source.device)
    desc = capi.ChConvDesc(n, h, w, c, r, s, padding[0], padding[1], stride[0], stride[1], ho, wo)
    capi.check("BlobChannelwiseConvolution", capi.load().nb200_blob_channelwise_convolution(
        _stream(), C.byref(desc), _ptr(_f32(source)), _ptr(_f32(filter)), _ptr(free_term), _ptr(result), act,
        float(act_param)))
    return result


def MobileNetV2Block(source, expand_filter, expand_free_term, channelwise_filter, channelwise_free_term, down_filter,
                     down_free_term, result=None, *, stride=1, residual=False, expand_act=ACT_RELU,
                     expand_act_param=6.0, channelwise_act=ACT_RELU, channelwise_act_param=6.0, scratch=None,
                     precision=PREC_3XTF32, one_kernel=False):
    """one_kernel: the block as a single kernel (nb200_mobilenetv2_block_fused; raises for shapes it does not cover)."""
    n, h, w, c_in = source.shape
    c_exp = expand_filter.shape[0]
    c_out = down_filter.shape[0]
    desc = capi.Mbv2Desc(n, h, w, c_in, c_exp, c_out, stride, int(residual), expand_act, channelwise_act,
                         float(expand_act_param), float(channelwise_act_param))
    lib = capi.load()
    need = lib.nb200_mobilenetv2_scratch_floats(C.byref(desc))
    if scratch is None or scratch.numel() < need:
        scratch = torch.empty(need, dtype=torch.float32, device=source.device)
    ho, wo = conv_output_size(h, 3, 1, stride), conv_output_size(w, 3, 1, stride)
    if result is None:
        result = torch.empty((n, ho, wo, c_out), dtype=torch.float32, device=source.device)
    entry = lib.nb200_mobilenetv2_block_fused if one_kernel else lib.nb200_mobilenetv2_block
    capi.check("MobileNetV2Block", entry(
        _stream(), C.byref(desc), _ptr(source), _ptr(expand_filter), _ptr(expand_free_term), _ptr(channelwise_filter),
        _ptr(channelwise_free_term), _ptr(down_filter), _ptr(down_free_term), _ptr(result), _ptr(scratch), precision))
    return result


def vector_op(op: str, first=None, second=None, scalar=None, value=0.0, result=None, count=None):
    """Elementwise family; `op` is one of capi.VEC_OPS.  `scalar` is a 1-element device tensor where the reference
    takes a handle (VectorMultiply, VectorReLU threshold, ...)."""
    done = _native().vector_op(VEC[op], first, second, scalar, value, result, count)
    if done is not None:
        return _checked("Vector" + op, done)
    ref = first if first is not None else result
    if result is None:
        result = torch.empty_like(ref)
    n = count if count is not None else result.numel()
    capi.check("Vector" + op, capi.load().nb200_vector_op(
        _stream(), VEC[op], _ptr(first), _ptr(second), _ptr(scalar), float(value), _ptr(result), n))
    return result


def VectorReLU(first, result=None, threshold=None):
    if threshold is None:
        threshold = torch.zeros(1, dtype=torch.float32, device=first.device)
    return vector_op("RELU", first, scalar=threshold, result=result)


def VectorAdd(first, second, result=None):
    return vector_op("ADD", first, second, result=result)


def AddVectorToMatrixRows(batch, matrix, vector, height, width, result=None):
    if result is None:
        result = torch.empty_like(matrix)
    capi.check("AddVectorToMatrixRows", capi.load().nb200_add_vector_to_matrix_rows(
        _stream(), batch, _ptr(matrix), _ptr(result), height, width, _ptr(vector)))
    return result


def AddVectorToMatrixColumns(matrix, vector, height, width, result=None):
    if result is None:
        result = torch.empty_like(matrix)
    capi.check("AddVectorToMatrixColumns", capi.load().nb200_add_vector_to_matrix_columns(
        _stream(), _ptr(matrix), _ptr(result), height, width, _ptr(vector)))
    return result


def SumMatrixRows(batch, matrix, height, width, result=None, add=False):
    if result is None:
        result = torch.empty((batch, width), dtype=torch.float32, device=matrix.device)
    capi.check("SumMatrixRows", capi.load().nb200_sum_matrix_rows(
        _stream(), batch, _ptr(result), _ptr(matrix), height, width, int(add)))
    return result


def SumMatrixColumns(matrix, height, width, result=None):
    if result is None:
        result = torch.empty(height, dtype=torch.float32, device=matrix.device)
    capi.check("SumMatrixColumns", capi.load().nb200_sum_matrix_columns(
        _stream(), _ptr(result), _ptr(matrix), height, width))
    return result


def MultiplyDiagMatrixByMatrix(diag, matrix, height, width, result=None):
    if result is None:
        result = torch.empty_like(matrix)
    capi.check("MultiplyDiagMatrixByMatrix", capi.load().nb200_multiply_diag_matrix_by_matrix(
        _stream(), _ptr(diag), height, _ptr(matrix), width, _ptr(result)))
    return result


def BatchMultiplyMatrixByDiagMatrix(batch, matrix, height, width, diag, diag_stride, result=None):
    if result is None:
        result = torch.empty_like(matrix)
    capi.check("BatchMultiplyMatrixByDiagMatrix", capi.load().nb200_multiply_matrix_by_diag_matrix(
        _stream(), batch, _ptr(matrix), height, width, _ptr(diag), diag_stride, _ptr(result)))
    return result


def MatrixSoftmaxByRows(matrix, height, width, result=None):
    if result is None:
        result = torch.empty_like(matrix)
    capi.check("MatrixSoftmaxByRows", capi.load().nb200_matrix_softmax_by_rows(
        _stream(), _ptr(matrix), height, width, _ptr(result)))
    return result


def MatrixSoftmaxByRowsFused(matrix, height, width, scale=None, row_bias=None, bias_rows=0, result=None):
    """softmax over the rows of (matrix * *scale + row_bias[h % bias_rows]): what the engine launches when an in-place
    VectorMultiply by a device scalar and an in-place AddVectorToMatrixRows precede an in-place MatrixSoftmaxByRows."""
    if result is None:
        result = torch.empty_like(matrix)
    capi.check("MatrixSoftmaxByRows (fused)", capi.load().nb200_matrix_softmax_by_rows_fused(
        _stream(), _ptr(matrix), height, width, _ptr(scale), _ptr(row_bias), bias_rows, _ptr(result)))
    return result


def TransposeMatrix(batch, first, height, medium, width, channels, result=None):
    done = _native().transpose(batch, first, height, medium, width, channels, result)
    if done is not None:
        return _checked("TransposeMatrix", done)
    if result is None:
        result = torch.empty_like(first)
    capi.check("TransposeMatrix", capi.load().nb200_transpose_matrix(
        _stream(), batch, _ptr(first), height, medium, width, channels, _ptr(result)))
    return result


def FindMaxValueInRows(matrix, height, width, with_indices=True):
    vals = torch.empty(height, dtype=torch.float32, device=matrix.device)
    idx = torch.empty(height, dtype=torch.int32, device=matrix.device) if with_indices else None
    capi.check("FindMaxValueInRows", capi.load().nb200_find_max_value_in_rows(
        _stream(), _ptr(matrix), height, width, _ptr(vals), _ptr(idx)))
    return vals, idx


def FindMaxValueInColumns(batch, matrix, height, width):
    vals = torch.empty((batch, width), dtype=torch.float32, device=matrix.device)
    idx = torch.empty((batch, width), dtype=torch.int32, device=matrix.device)
    capi.check("FindMaxValueInColumns", capi.load().nb200_find_max_value_in_columns(
        _stream(), batch, _ptr(matrix), height, width, _ptr(vals), _ptr(idx)))
    return vals, idx


def BlobMaxPooling(source, filter_size, stride, result=None, with_indices=False):
    n, h, w, c = source.shape
    ho, wo = (h - filter_size[0]) // stride[0] + 1, (w - filter_size[1]) // stride[1] + 1
    if result is None:
        result = torch.empty((n, ho, wo, c), dtype=torch.float32, device=source.device)
    idx = torch.empty((n, ho, wo, c), dtype=torch.int32, device=source.device) if with_indices else None
    capi.check("BlobMaxPooling", capi.load().nb200_blob_max_pooling(
        _stream(), n, h, w, c, filter_size[0], filter_size[1], stride[0], stride[1], _ptr(source), _ptr(result),
        _ptr(idx)))
    return (result, idx) if with_indices else result


def AttentionScoresValues(q, kt, v, scale=None, mask=None, precision=PREC_3XTF32):
    """softmax(scale * q @ kt + mask) @ v per batch entry; q [b, sq, d], kt [b, d, st], v [b, st, d]; scale: a 1-element
    device tensor or None; mask [sq, st] or None."""
    b, sq, d = q.shape
    st = kt.shape[2]
    out = torch.empty((b, sq, d), dtype=torch.float32, device=q.device)
    capi.check("AttentionScoresValues", capi.load().nb200_attention_scores_values(
        _stream(), b, _ptr(q), _ptr(kt), _ptr(v), sq, d, st, _ptr(scale), _ptr(mask), _ptr(out), precision))
    return out


def BlobMaxPoolingPadded(source, deltas, default_value, filter_size, stride, result=None):
    """BlobResizeImage (constant padding; deltas = left, right, top, bottom) + BlobMaxPooling as one pass."""
    n, h, w, c = source.shape
    left, right, top, bottom = deltas
    ho = (h + top + bottom - filter_size[0]) // stride[0] + 1
    wo = (w + left + right - filter_size[1]) // stride[1] + 1
    if result is None:
        result = torch.empty((n, ho, wo, c), dtype=torch.float32, device=source.device)
    capi.check("BlobMaxPoolingPadded", capi.load().nb200_blob_max_pooling_padded(
        _stream(), n, h, w, c, left, right, top, bottom, float(default_value), filter_size[0], filter_size[1], stride[0],
        stride[1], _ptr(source), _ptr(result)))
    return result


def BlobMeanPooling(source, filter_size, stride, result=None):
    n, h, w, c = source.shape
    ho, wo = (h - filter_size[0]) // stride[0] + 1, (w - filter_size[1]) // stride[1] + 1
    if result is None:
        result = torch.empty((n, ho, wo, c), dtype=torch.float32, device=source.device)
    capi.check("BlobMeanPooling", capi.load().nb200_blob_mean_pooling(
        _stream(), n, h, w, c, filter_size[0], filter_size[1], stride[0], stride[1], _ptr(source), _ptr(result)))
    return result


def BlobResizeImage(source, delta_left, delta_right, delta_top, delta_bottom, padding=0, default_value=0.0,
                    result=None):
    n, h, w, c = source.shape
    if result is None:
        result = torch.empty((n, h + delta_top + delta_bottom, w + delta_left + delta_right, c), dtype=torch.float32,
                             device=source.device)
    capi.check("BlobResizeImage", capi.load().nb200_blob_resize_image(
        _stream(), n, h, w, c, delta_left, delta_right, delta_top, delta_bottom, padding, float(default_value),
        _ptr(source), _ptr(result)))
    return result


# ---- operators of language models: fp32, fp16 and bf16 data, fp32 sums -----------------------------------------------

_TYPES = {torch.float32: capi.TYPE_FP32, torch.float16: capi.TYPE_FP16, torch.bfloat16: capi.TYPE_BF16}


def _typed(t: torch.Tensor) -> int:
    assert t.dtype in _TYPES, f"fp32, fp16 or bf16 tensors only, not {t.dtype}"
    return _TYPES[t.dtype]


def _device_of(*tensors) -> torch.device:
    """The one device that all of them (None left out) are on."""
    assert not any(t is not None and t.is_neg() for t in tensors), "tensors that hold their own values, no negated views"
    devices = {t.device for t in tensors if t is not None}
    assert len(devices) == 1 and next(iter(devices)).type == "cuda", "tensors on one CUDA device only"
    return next(iter(devices))


def _current(device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _matrix(t: torch.Tensor) -> tuple[int, int, int]:
    """Rows, width and row size of a tensor seen as a matrix of its last dimension; a 2-D one may be a view of some
    columns or of every n-th row."""
    assert t.dim() >= 1 and t.shape[-1] >= 1, "rows of at least one element"
    width = t.shape[-1]
    if t.dim() == 2 and t.shape[0] > 1:
        assert (width == 1 or t.stride(1) == 1) and t.stride(0) >= width, "rows of adjacent elements that do not overlap"
        return t.shape[0], width, t.stride(0)
    assert t.is_contiguous(), "contiguous tensors, or matrices of contiguous rows"
    return t.numel() // width, width, width


def _vector(t: torch.Tensor | None, count: int, *types) -> int | None:
    """Pointer of an optional contiguous vector with `count` elements of one of the types."""
    if t is None:
        return None
    assert t.numel() == count and t.is_contiguous() and t.dtype in types, f"{count} contiguous elements of {types}"
    return t.data_ptr()


def LayerNormalization(source, scale=None, free_term=None, *, epsilon=1e-5, result=None):
    """The rows of `source` [..., width], each less its mean and over its deviation, times `scale` plus `free_term`.  Returns
    (result, mean, inverse_deviation); the last two are what the backward pass takes, fp32, one per row.  scale and
    free_term have `width` elements, both of the source's type or both fp32; None stands for ones and zeros.  `result` may
    be `source`."""
    done = _native().layer_normalization(source, scale, free_term, epsilon, result)
    if done is not None:
        return _checked("LayerNormalization", done)
    height, width, row = _matrix(source)
    code, parameter = _typed(source), next((p.dtype for p in (scale, free_term) if p is not None), source.dtype)
    assert parameter in (source.dtype, torch.float32), "parameters of the rows' type or fp32"
    if result is None:
        result = torch.empty(source.shape, dtype=source.dtype, device=source.device)
    assert result.shape == source.shape and result.dtype == source.dtype, "a result like the source"
    device = _device_of(source, scale, free_term, result)
    scale_at, free_at = _vector(scale, width, parameter), _vector(free_term, width, parameter)
    mean, inverse = torch.empty((2, *source.shape[:-1]), dtype=torch.float32, device=device).unbind()
    with torch.cuda.device(device):
        capi.check("LayerNormalization", capi.load().nb200_layer_normalization(
            _current(device), code, _TYPES[parameter], source.data_ptr(), height, width, row, scale_at, free_at, float(epsilon),
            result.data_ptr(), _matrix(result)[2], mean.data_ptr(), inverse.data_ptr()))
    return result, mean, inverse


def LayerNormalizationBackward(result_diff, source, mean, inverse_deviation, scale=None, *, source_diff=None,
                               parameters=True, parameter_type=None):
    """The gradients of LayerNormalization: (source_diff, scale_diff, free_term_diff) from the result's, what went in and
    the two vectors that the forward pass returned.  The parameters' gradients are of the scale's type (without a scale
    `parameter_type`, or the source's); None with parameters=False.  `source_diff` may be `result_diff`."""
    done = _native().layer_normalization_backward(result_diff, source, mean, inverse_deviation, scale, source_diff,
                                                   parameters)
    if done is not None:
        return _checked("LayerNormalizationBackward", done)
    height, width, row = _matrix(source)
    code = _typed(source)
    parameter = scale.dtype if scale is not None else parameter_type or source.dtype
    assert parameter in (source.dtype, torch.float32), "parameters of the rows' type or fp32"
    if source_diff is None:
        source_diff = torch.empty(source.shape, dtype=source.dtype, device=source.device)
    for t in (result_diff, source_diff):
        assert t.shape == source.shape and t.dtype == source.dtype, "gradients like the source"
    device = _device_of(result_diff, source, mean, inverse_deviation, scale, source_diff)
    mean_at, inverse_at = _vector(mean, height, torch.float32), _vector(inverse_deviation, height, torch.float32)
    scale_at = _vector(scale, width, parameter)
    lib = capi.load()
    scale_diff = free_diff = scratch = None
    with torch.cuda.device(device):
        if parameters:
            scale_diff, free_diff = (torch.empty(width, dtype=parameter, device=device) for _ in range(2))
            need = lib.nb200_layer_normalization_backward_scratch_floats(code, height, width)
            scratch = torch.empty(need, dtype=torch.float32, device=device)
        capi.check("LayerNormalizationBackward", lib.nb200_layer_normalization_backward(
            _current(device), code, _TYPES[parameter], result_diff.data_ptr(), _matrix(result_diff)[2], source.data_ptr(), height,
            width, row, scale_at, mean_at, inverse_at, source_diff.data_ptr(), _matrix(source_diff)[2], _ptr(scale_diff),
            _ptr(free_diff), _ptr(scratch)))
    return source_diff, scale_diff, free_diff


def _steps(t: torch.Tensor, shape, dtype) -> tuple[int, int]:
    """Strides of a [batch, length, channels] operand with adjacent channels; expanded ones repeat."""
    assert t.shape == shape and t.dtype == dtype, f"{list(shape)} of {dtype}"
    assert shape[2] <= 1 or t.stride(2) == 1, "adjacent channels"
    return (t.stride(0) if shape[0] > 1 else 0), (t.stride(1) if shape[1] > 1 else 0)


def _recurrence_desc(update, forget, input):
    assert update.dim() == 3, "[batch, length, channels]"
    shape, dtype = update.shape, update.dtype
    return capi.RecurrenceDesc(*shape, *_steps(update, shape, dtype), *_steps(forget, shape, dtype),
                               *(_steps(input, shape, dtype) if input is not None else (0, 0)))


def GatedRecurrence(update, forget, input=None, *, initial_state=None, lengths=None, result=None, final_state=None):
    """h[t] = sigmoid(forget[t]) h[t-1] + u[t] update[t] over [batch, length, channels], u = sigmoid(input) or, without
    input gates, 1 - sigmoid(forget): QrnnIfPooling and QrnnFPooling with the gates' sigmoid inside.  Returns (result,
    final_state): every h[t] in the update's type, and the last state, fp32 [batch, channels].  initial_state is fp32 too
    (None: zeros); `final_state` may be the same tensor, as when tokens are served one at a time.  lengths (int32 [batch])
    ends sequences early: behind their end the result is zero and the state stays.  The three inputs may be strided views or
    expanded; channels are adjacent.  At most 65535 sequences."""
    done = _native().gated_recurrence(update, forget, input, initial_state, lengths, result, final_state)
    if done is not None:
        return _checked("GatedRecurrence", done)
    desc, code = _recurrence_desc(update, forget, input), _typed(update)
    batch, length, channels = update.shape
    if result is None:
        result = torch.empty(update.shape, dtype=update.dtype, device=update.device)
    if final_state is None:
        final_state = torch.empty((batch, channels), dtype=torch.float32, device=update.device)
    assert result.shape == update.shape and result.dtype == update.dtype and result.is_contiguous(), "a dense result like the update"
    device = _device_of(update, forget, input, initial_state, lengths, result, final_state)
    states = _vector(initial_state, batch * channels, torch.float32), _vector(final_state, batch * channels, torch.float32)
    lengths_at = _vector(lengths, batch, torch.int32)
    with torch.cuda.device(device):
        capi.check("GatedRecurrence", capi.load().nb200_gated_recurrence(
            _current(device), code, C.byref(desc), update.data_ptr(), forget.data_ptr(),
            None if input is None else input.data_ptr(), states[0], lengths_at, result.data_ptr(), states[1]))
    return result, final_state


def GatedRecurrenceBackward(result_diff, result, update, forget, input=None, *, initial_state=None, final_state_diff=None,
                            lengths=None):
    """The gradients of GatedRecurrence: (update_diff, forget_diff, input_diff, initial_state_diff); input_diff is None
    without input gates.  `result` is what the forward pass returned (the states themselves are fp32 here too: those of 16-bit
    types are formed again from the inputs); final_state_diff (fp32, None: zeros) is the gradient of the last state.  Gradients are dense, one for every element that an expanded input stands for, and zero behind a
    sequence's end."""
    done = _native().gated_recurrence_backward(result_diff, result, update, forget, input, initial_state, final_state_diff, lengths)
    if done is not None:
        return _checked("GatedRecurrenceBackward", done)
    desc, code = _recurrence_desc(update, forget, input), _typed(update)
    batch, length, channels = update.shape
    diff_strides = _steps(result_diff, update.shape, update.dtype)
    assert result.shape == update.shape and result.dtype == update.dtype and result.is_contiguous(), "the forward pass's result"
    device = _device_of(result_diff, result, update, forget, input, initial_state, final_state_diff, lengths)
    states = _vector(initial_state, batch * channels, torch.float32), _vector(final_state_diff, batch * channels, torch.float32)
    lengths_at = _vector(lengths, batch, torch.int32)
    update_diff, forget_diff = torch.empty_like(result), torch.empty_like(result)
    input_diff = None if input is None else torch.empty_like(result)
    initial_diff = torch.empty((batch, channels), dtype=torch.float32, device=device)
    with torch.cuda.device(device):
        capi.check("GatedRecurrenceBackward", capi.load().nb200_gated_recurrence_backward(
            _current(device), code, C.byref(desc), result_diff.data_ptr(), *diff_strides, result.data_ptr(), update.data_ptr(),
            forget.data_ptr(), None if input is None else input.data_ptr(), states[0], states[1], lengths_at,
            update_diff.data_ptr(), forget_diff.data_ptr(), _ptr(input_diff), initial_diff.data_ptr()))
    return update_diff, forget_diff, input_diff, initial_diff


def _teacher(logits, teacher_logits, teacher_indices, rows, temperature):
    assert teacher_logits.shape == teacher_indices.shape and teacher_logits.shape[:-1] == logits.shape[:-1], \
        "the kept logits and their columns, for every row"
    assert teacher_logits.dtype in (logits.dtype, torch.float32), "a teacher of the logits' type or fp32"
    assert 0.0 < temperature < float("inf"), "a positive temperature"
    kept = teacher_logits.shape[-1]
    return kept, _vector(teacher_logits, rows * kept, teacher_logits.dtype), _vector(teacher_indices, rows * kept, torch.int32)


def DistillationLoss(logits, teacher_logits, teacher_indices, *, temperature=1.0):
    """temperature^2 times the divergence of a student's rows of `logits` [..., vocabulary] from a teacher of which each row
    kept some top logits: teacher_logits and teacher_indices (int32) [..., kept], at most 1024 of them, renormalised among
    themselves.  An index outside the vocabulary marks an entry that is not used; rows without one have loss zero.
    Returns (loss, log_sum), fp32, one per row; log_sum, of logits / temperature, is what the backward pass takes."""
    done = _native().distillation_loss(logits, teacher_logits, teacher_indices, temperature)
    if done is not None:
        return _checked("DistillationLoss", done)
    rows, vocabulary, row = _matrix(logits)
    code = _typed(logits)
    kept, teacher_at, indices_at = _teacher(logits, teacher_logits, teacher_indices, rows, temperature)
    device = _device_of(logits, teacher_logits, teacher_indices)
    loss, log_sum = torch.empty((2, *logits.shape[:-1]), dtype=torch.float32, device=device).unbind()
    with torch.cuda.device(device):
        capi.check("DistillationLoss", capi.load().nb200_distillation_loss(
            _current(device), code, _TYPES[teacher_logits.dtype], logits.data_ptr(), rows, vocabulary, row, teacher_at, indices_at,
            kept, float(temperature), loss.data_ptr(), log_sum.data_ptr()))
    return loss, log_sum


def DistillationLossBackward(loss_diff, logits, teacher_logits, teacher_indices, log_sum, *, temperature=1.0, result=None):
    """The gradient of DistillationLoss by the logits, from that of each row's loss (fp32) and the log_sum of the forward
    pass.  `result` may be `logits`, which the gradient then replaces."""
    done = _native().distillation_loss_backward(loss_diff, logits, teacher_logits, teacher_indices, log_sum, temperature, result)
    if done is not None:
        return _checked("DistillationLossBackward", done)
    rows, vocabulary, row = _matrix(logits)
    code = _typed(logits)
    kept, teacher_at, indices_at = _teacher(logits, teacher_logits, teacher_indices, rows, temperature)
    if result is None:
        result = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    assert result.shape == logits.shape and result.dtype == logits.dtype, "a gradient like the logits"
    device = _device_of(loss_diff, logits, teacher_logits, teacher_indices, log_sum, result)
    diff_at, sum_at = _vector(loss_diff, rows, torch.float32), _vector(log_sum, rows, torch.float32)
    with torch.cuda.device(device):
        capi.check("DistillationLossBackward", capi.load().nb200_distillation_loss_backward(
            _current(device), code, _TYPES[teacher_logits.dtype], diff_at, logits.data_ptr(), rows, vocabulary, row, teacher_at,
            indices_at, kept, float(temperature), sum_at, result.data_ptr(), _matrix(result)[2]))
    return result


def _head(hidden, weights, labels):
    rows, width, row = _matrix(hidden)
    assert weights.dim() == 2 and weights.shape[1] == width and weights.dtype == hidden.dtype, \
        f"weights [vocabulary, {width}] of the hidden rows' type"
    vocabulary, _, weights_row = _matrix(weights)
    assert vocabulary >= 1, "a vocabulary"
    assert labels.shape == hidden.shape[:-1], "a label for every row"
    return _typed(hidden), rows, width, row, vocabulary, weights_row


def _head_scratch(code, hidden, rows, width, row, weights, vocabulary, weights_row, backward):
    need = capi.load().nb200_vocabulary_cross_entropy_scratch_bytes(code, hidden.data_ptr(), rows, width, row, weights.data_ptr(),
                                                                    vocabulary, weights_row, int(backward))
    return torch.empty(need, dtype=torch.uint8, device=hidden.device)


def VocabularyCrossEntropy(hidden, weights, labels):
    """Softmax cross entropy of the logits hidden @ weights^T against labels (int32), without keeping the logits: hidden
    [..., width], weights [vocabulary, width], labels [...].  Returns (loss, log_sum), fp32, one per row; log_sum is what the
    backward pass takes.  A label outside the vocabulary marks a row without a target (padding, a prompt): loss zero."""
    done = _native().vocabulary_cross_entropy(hidden, weights, labels)
    if done is not None:
        return _checked("VocabularyCrossEntropy", done)
    code, rows, width, row, vocabulary, weights_row = _head(hidden, weights, labels)
    device = _device_of(hidden, weights, labels)
    labels_at = _vector(labels, rows, torch.int32)
    loss, log_sum = torch.empty((2, *labels.shape), dtype=torch.float32, device=device).unbind()
    with torch.cuda.device(device):
        scratch = _head_scratch(code, hidden, rows, width, row, weights, vocabulary, weights_row, False)
        capi.check("VocabularyCrossEntropy", capi.load().nb200_vocabulary_cross_entropy(
            _current(device), code, hidden.data_ptr(), rows, width, row, weights.data_ptr(), vocabulary, weights_row, labels_at,
            loss.data_ptr(), log_sum.data_ptr(), scratch.data_ptr()))
    return loss, log_sum


def VocabularyCrossEntropyBackward(loss_diff, hidden, weights, labels, log_sum, *, hidden_diff=True, weights_diff=True):
    """The gradients of VocabularyCrossEntropy by hidden and weights, from that of each row's loss (fp32) and the forward
    pass's log_sum.  hidden_diff and weights_diff: True for a new tensor, the tensor to write, or False or None where that
    gradient is not wanted (None comes back).  Rows without a target have no gradient."""
    done = _native().vocabulary_cross_entropy_backward(loss_diff, hidden, weights, labels, log_sum, hidden_diff, weights_diff)
    if done is not None:
        return _checked("VocabularyCrossEntropyBackward", done)
    code, rows, width, row, vocabulary, weights_row = _head(hidden, weights, labels)
    device = _device_of(loss_diff, hidden, weights, labels, log_sum)
    pointers = (_vector(loss_diff, rows, torch.float32), _vector(labels, rows, torch.int32), _vector(log_sum, rows, torch.float32))
    diffs, places = [], []
    for wanted, like in ((hidden_diff, hidden), (weights_diff, weights)):
        diff = torch.empty(like.shape, dtype=like.dtype, device=device) if wanted is True else None if wanted is False else wanted
        diffs.append(diff)
        if diff is not None:
            assert diff.shape == like.shape and diff.dtype == like.dtype and diff.device == device and not diff.is_neg(), \
                "gradients like their operands"
        places += (None, 0) if diff is None else (diff.data_ptr(), _matrix(diff)[2])
    with torch.cuda.device(device):
        scratch = _head_scratch(code, hidden, rows, width, row, weights, vocabulary, weights_row, True)
        capi.check("VocabularyCrossEntropyBackward", capi.load().nb200_vocabulary_cross_entropy_backward(
            _current(device), code, pointers[0], hidden.data_ptr(), rows, width, row, weights.data_ptr(), vocabulary, weights_row,
            pointers[1], pointers[2], *places, scratch.data_ptr()))
    return tuple(diffs)
