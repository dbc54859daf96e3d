"""Host-side mirror of the reference's quantized-Dense operator interface over torch
device tensors.  Names, argument meaning and error behaviour follow

* ``nn.QuantizedDense``   ml/nn/quantized_dense.go:31-57
* ``nn.QuantizedGather``  ml/nn/quantized_gather.go:30-43
* ``ggml.Dequantize``     ml/ggml/dequant.go:39-54
* ``graph.Quantization``  core/graph/fused_ops.go:18-48
* ``activation.Type.ToBackend``  ml/layers/activation/activation.go:58-75

torch only supplies device memory and the current stream; all arithmetic runs in
libgomlx_hipq.so.  There is no CPU path: tensors must live on the GPU.

The operators of a decode loop first try the same steps in native code (``_lib.fast``,
csrc/binding.cpp; bound by the first of these calls, so used from a process's second one on); it
returns None for whatever it does not take, and the Python steps below then run or raise.
"""
from __future__ import annotations

import enum
from dataclasses import dataclass

import torch

from . import _lib, ggml


class QuantizationScheme(enum.IntEnum):
    """compute.QuantizationScheme; only GGML is on this path."""
    LINEAR = 0
    NF4 = 1
    GGML = 2


class Activation(enum.IntEnum):
    """activation.Type of the reference (ml/layers/activation/activation.go:30-54)."""
    NONE = 0
    RELU = 1
    SIGMOID = 2
    HARD_SIGMOID = 3
    LEAKY_RELU = 4
    SELU = 5
    SWISH = 6
    HARD_SWISH = 7
    SILU = 8
    TANH = 9
    GELU = 10
    GELU_APPROX = 11
    SWIGLU = 12

    def to_backend(self) -> int:
        """activation.Type.ToBackend: types without a backend enum map to NONE, and both
        GELU flavours map to the single backend Gelu (activation.go:58-75)."""
        return {
            Activation.NONE: 0, Activation.GELU: 1, Activation.GELU_APPROX: 1, Activation.RELU: 2,
            Activation.SWISH: 3, Activation.SILU: 3, Activation.HARD_SWISH: 4, Activation.TANH: 5,
        }.get(self, 0)


_NO_ACTIVATION = Activation.NONE  # (a member looked up through its class costs every call 0.05 us)


@dataclass
class Quantization:
    """graph.Quantization (core/graph/fused_ops.go:18-48).  For GGML only scheme and
    ggml_type are used; the scales live inside the blocks."""
    scheme: QuantizationScheme = QuantizationScheme.GGML
    ggml_type: int = ggml.Q8_0
    scale: object = None
    zero_point: object = None
    block_axis: int = 0
    block_size: int = 0


def _init(device: int) -> None:
    _lib.init(device)
    _lib.bind_fast(Activation)


def _stream_ptr(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


def _require_cuda(name: str, t: torch.Tensor) -> None:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a GPU tensor: this backend has no CPU path")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _weights_2d(weights: torch.Tensor) -> None:
    if weights.dtype != torch.uint8 or weights.dim() != 2:
        raise ValueError("weights must be a Uint8 [N, bytesPerRow] tensor of native GGML blocks")


def dequantize(weights: torch.Tensor, ggml_type: int) -> torch.Tensor:
    """ggml.Dequantize: [N, bytesPerRow] uint8 -> [N, K] float32, bit-exact."""
    if _lib.fast is not None and (out := _lib.fast.dequantize(weights, ggml_type)) is not None:
        return out
    _require_cuda("weights", weights)
    _weights_2d(weights)
    _init(weights.device.index or 0)
    N, rb = weights.shape
    bpb = ggml.bytes_per_block(ggml_type)
    if rb % bpb:
        raise ValueError(f"row of {rb} bytes is not a whole number of {bpb}-byte blocks")
    K = rb // bpb * ggml.values_per_block(ggml_type)
    out = torch.empty((N, K), dtype=torch.float32, device=weights.device)
    _lib.check(_lib.lib().gq_dequantize(ggml_type, weights.data_ptr(), N, K, out.data_ptr(), _stream_ptr(weights)))
    return out


@dataclass
class RMSNorm:
    """Configuration of norm.RMSNorm over the last axis (ml/layers/norm/rmsnorm.go:38-76): ``gain`` is the
    learned scale [K] (None = WithScale(false)), ``epsilon`` WithEpsilon (default 1e-6), ``scale_offset``
    WithScaleOffset (Gemma adds 1.0 to the scale)."""
    gain: torch.Tensor | None = None
    epsilon: float = 1e-6
    scale_offset: float = 0.0

    def _desc(self, K: int):
        if self.gain is not None:
            _require_cuda("gain", self.gain)
            if self.gain.dtype != torch.float32 or tuple(self.gain.shape) != (K,):
                raise ValueError(f"gain must be a float32 [{K}] tensor")
        return _lib.RmsNormDesc(None if self.gain is None else self.gain.data_ptr(), self.epsilon, self.scale_offset)


def rms_norm(x: torch.Tensor, norm: RMSNorm) -> torch.Tensor:
    """RMSNormBuilder.Done (ml/layers/norm/rmsnorm.go:78-113) over the last axis of a float32 tensor."""
    _require_cuda("x", x)
    if x.dtype != torch.float32:
        raise _lib.NotImplementedByBackend(_lib.ERR_NOT_IMPLEMENTED, f"rms_norm: dtype {x.dtype} is not implemented")
    K = x.shape[-1]
    d = norm._desc(K)
    _init(x.device.index or 0)
    y = torch.empty_like(x)
    _lib.check(_lib.lib().gq_rmsnorm_f32(x.data_ptr(), x.numel() // K if K else 0, K, d.dGain, d.eps, d.gain_offset, y.data_ptr(),
                                         _stream_ptr(x)))
    return y


def gated_feed_forward(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, quant: Quantization, activation: Activation,
                       bias_gate: torch.Tensor | None = None, bias_up: torch.Tensor | None = None,
                       norm: RMSNorm | None = None) -> torch.Tensor:
    """The front of a gated feed-forward block (ml/zoo/transformer/transformer.go:1276-1287):
    ``activation(dense(xn, w_gate)) * dense(xn, w_up)`` with ``xn = rms_norm(x)`` when ``norm`` is given.
    x: [batch..., K] float32 or bfloat16 (gain, biases and the result stay float32); both weights [N, bytesPerRow] uint8 of one GGML type."""
    if _lib.fast is not None and (y := _lib.fast.gated(x, w_gate, w_up, quant, activation, bias_gate, bias_up, norm)) is not None:
        return y
    if quant is None or quant.scheme != QuantizationScheme.GGML:
        raise _lib.NotImplementedByBackend(_lib.ERR_NOT_IMPLEMENTED, "only the GGML scheme is on this path")
    for name, t in (("x", x), ("w_gate", w_gate), ("w_up", w_up)):
        _require_cuda(name, t)
    _weights_2d(w_gate)
    _weights_2d(w_up)
    if w_gate.shape != w_up.shape:
        raise ValueError(f"gate and up weights differ in shape: {tuple(w_gate.shape)} vs {tuple(w_up.shape)}")
    if x.dtype not in (torch.float32, torch.bfloat16):
        raise _lib.NotImplementedByBackend(_lib.ERR_NOT_IMPLEMENTED, f"gated_feed_forward: dtype {x.dtype} is not implemented")
    xd = _lib.F32 if x.dtype == torch.float32 else _lib.BF16
    import ctypes
    L = _lib.lib()
    N, rb = w_gate.shape
    K_in = x.shape[-1]
    M = x.numel() // K_in if K_in else 0
    K = ctypes.c_int64(0)
    for b in (bias_gate, bias_up):
        blen = -1
        if b is not None:
            _require_cuda("bias", b)
            if b.dtype != torch.float32 or b.dim() != 1:
                raise ValueError("bias must be a float32 [N] tensor")
            blen = b.shape[0]
        _lib.check(L.gq_qdense_check(quant.ggml_type, xd, M, K_in, N, rb, blen, activation.to_backend(), ctypes.byref(K)))
    d = None if norm is None else norm._desc(K.value)
    _init(x.device.index or 0)
    y = torch.empty(x.shape[:-1] + (N,), dtype=torch.float32, device=x.device)
    fn = L.gq_qdense_gated_f32 if xd == _lib.F32 else L.gq_qdense_gated_bf16
    _lib.check(fn(quant.ggml_type, x.data_ptr(), M, K.value, None if d is None else ctypes.byref(d),
                                     w_gate.data_ptr(), None if bias_gate is None else bias_gate.data_ptr(), w_up.data_ptr(),
                                     None if bias_up is None else bias_up.data_ptr(), N, activation.to_backend(), y.data_ptr(),
                                     _stream_ptr(x)))
    return y


def quantized_dense(x: torch.Tensor, weights: torch.Tensor, quant: Quantization, bias: torch.Tensor | None = None,
                    *optional_activation: Activation, norm: RMSNorm | None = None,
                    residual: torch.Tensor | None = None) -> torch.Tensor:
    """nn.QuantizedDense for the GGML scheme: y = activation(x @ dequant(weights)^T + bias).

    x: [batch..., K] float32 or bfloat16; weights: [N, bytesPerRow] uint8; bias: [N] float32.
    Returns [batch..., N] float32.  ``norm`` applies an RMS normalisation to x first and ``residual``
    ([batch..., N] float32) is added to the result (gain and residual are float32 also for bfloat16 x): Model.normalize followed by a
    projection and Add(residual, ...) after it, ml/zoo/transformer/transformer.go:1099-1101, 1045, 1055.
    """
    if _lib.fast is not None and len(optional_activation) <= 1:
        y = _lib.fast.dense(x, weights, quant, bias, optional_activation[0] if optional_activation else _NO_ACTIVATION, norm, residual)
        if y is not None:
            return y
    if len(optional_activation) > 1:
        raise ValueError(f"quantized_dense can only take one optional activation, got {optional_activation}")
    act = optional_activation[0] if optional_activation else Activation.NONE
    if quant is None:
        raise ValueError("quant must not be None")  # core/graph/fused_ops.go:198-200
    if quant.scheme != QuantizationScheme.GGML:
        raise _lib.NotImplementedByBackend(_lib.ERR_NOT_IMPLEMENTED,
                                           f"scheme {quant.scheme.name} is outside this backend (GGML only)")
    _require_cuda("x", x)
    _require_cuda("weights", weights)
    _weights_2d(weights)
    if x.dtype == torch.float32:
        xd = _lib.F32
    elif x.dtype == torch.bfloat16:
        xd = _lib.BF16
    else:
        raise _lib.NotImplementedByBackend(_lib.ERR_NOT_IMPLEMENTED, f"activation dtype {x.dtype} is not implemented")
    L = _lib.lib()
    N, rb = weights.shape
    K_in = x.shape[-1]
    M = x.numel() // K_in if K_in else 0
    blen = -1
    if bias is not None:
        _require_cuda("bias", bias)
        if bias.dtype != torch.float32 or bias.dim() != 1:
            raise ValueError("bias must be a float32 [N] tensor")
        blen = bias.shape[0]
    import ctypes
    K = ctypes.c_int64(0)
    _lib.check(L.gq_qdense_check(quant.ggml_type, xd, M, K_in, N, rb, blen, act.to_backend(), ctypes.byref(K)))
    _init(x.device.index or 0)
    y = torch.empty(x.shape[:-1] + (N,), dtype=torch.float32, device=x.device)
    if norm is not None or residual is not None:
        d = None if norm is None else norm._desc(K.value)
        if residual is not None:
            _require_cuda("residual", residual)
            if residual.dtype != torch.float32 or tuple(residual.shape) != tuple(y.shape):
                raise ValueError(f"residual must be a float32 tensor of shape {tuple(y.shape)}")
        block = L.gq_qdense_block_f32 if xd == _lib.F32 else L.gq_qdense_block_bf16
        _lib.check(block(quant.ggml_type, x.data_ptr(), M, K.value, None if d is None else ctypes.byref(d),
                                         weights.data_ptr(), N, None if bias is None else bias.data_ptr(), act.to_backend(),
                                         None if residual is None else residual.data_ptr(), y.data_ptr(), _stream_ptr(x)))
        return y
    fn = L.gq_qdense_f32 if xd == _lib.F32 else L.gq_qdense_bf16
    _lib.check(fn(quant.ggml_type, x.data_ptr(), M, K.value, weights.data_ptr(), N,
                  None if bias is None else bias.data_ptr(), act.to_backend(), y.data_ptr(), _stream_ptr(x)))
    return y


def quantized_gather(table: torch.Tensor, indices: torch.Tensor, quant: Quantization) -> torch.Tensor:
    """nn.QuantizedGather: indices [batch..., 1] (int32) -> [batch..., K] float32 rows of the
    dequantised table.  An out-of-range index raises IndexError: the call waits for the stream, and returns with the rows written."""
    if _lib.fast is not None and (out := _lib.fast.gather(table, indices, quant)) is not None:
        return out
    if quant.scheme != QuantizationScheme.GGML:
        raise ValueError("quantized_gather: only the GGML scheme is supported")  # quantized_gather.go:31-33
    _require_cuda("table", table)
    _require_cuda("indices", indices)
    _weights_2d(table)
    if indices.dim() < 1 or indices.shape[-1] != 1:
        raise ValueError("indices must have last dimension 1")
    idx = indices.to(torch.int32).contiguous()
    _init(table.device.index or 0)
    vocab, rb = table.shape
    bpb = ggml.bytes_per_block(quant.ggml_type)
    if rb % bpb:
        raise ValueError(f"row of {rb} bytes is not a whole number of {bpb}-byte blocks")
    K = rb // bpb * ggml.values_per_block(quant.ggml_type)
    count = idx.numel()
    out = torch.empty(tuple(indices.shape[:-1]) + (K,), dtype=torch.float32, device=table.device)
    flag = torch.zeros(1, dtype=torch.int32, device=table.device)
    _lib.check(_lib.lib().gq_embedding_lookup(quant.ggml_type, table.data_ptr(), vocab, K, idx.data_ptr(), count,
                                              out.data_ptr(), flag.data_ptr(), _stream_ptr(table)))
    if count and int(flag.item()):
        raise IndexError("quantized_gather: index out of range")
    return out


def quantized_dense_batch(problems, norm: RMSNorm | None = None) -> list:
    """Several independent nn.QuantizedDense calls submitted together (gq_qdense_f32_batch); with
    ``norm`` every problem's activations are RMS-normalised first (the q/k/v projections behind a
    layer's input norm, gq_qdense_norm_f32_batch).

    ``problems`` is a sequence of ``(x, weights, quant, bias, activation)`` tuples with float32
    activations (with ``norm``: all float32 or all bfloat16); returns the list of outputs.  Problems of one GGML type and one batch size of
    up to 8 rows share a kernel launch, as do projections of one ``x`` of up to 16 rows and, behind a norm or in Q4_K, of more.  Results equal those of separate calls to
    the rounding of the activations, not bit for bit: a list may take a kernel that its members alone do not (batches of 1 and 2 rows take
    the same; from 3 rows the difference stays within 1e-4 of a row's 2-norm, for Q4_K from 9 rows and any format from 17 within 1.2e-3).
    """
    if _lib.fast is not None and (outs := _lib.fast.batch(problems, norm)) is not None:
        return outs
    import ctypes
    L = _lib.lib()
    descs = (_lib.DenseDesc * len(problems))()
    outs = []
    for i, (x, weights, quant, bias, act) in enumerate(problems):
        act = Activation.NONE if act is None else act
        if quant is None or quant.scheme != QuantizationScheme.GGML:
            raise _lib.NotImplementedByBackend(_lib.ERR_NOT_IMPLEMENTED, "only the GGML scheme is on this path")
        _require_cuda("x", x)
        _require_cuda("weights", weights)
        _weights_2d(weights)
        bf16 = norm is not None and x.dtype == torch.bfloat16 and all(p[0].dtype == torch.bfloat16 for p in problems)
        if x.dtype != torch.float32 and not bf16:
            raise _lib.NotImplementedByBackend(_lib.ERR_NOT_IMPLEMENTED, "batched submission takes float32 activations "
                                               "(behind a shared normalisation: all float32 or all bfloat16)")
        N, rb = weights.shape
        K_in = x.shape[-1]
        M = x.numel() // K_in if K_in else 0
        blen = -1
        if bias is not None:
            _require_cuda("bias", bias)
            blen = bias.shape[0]
        K = ctypes.c_int64(0)
        _lib.check(L.gq_qdense_check(quant.ggml_type, _lib.BF16 if bf16 else _lib.F32, M, K_in, N, rb, blen, act.to_backend(), ctypes.byref(K)))
        y = torch.empty(x.shape[:-1] + (N,), dtype=torch.float32, device=x.device)
        outs.append(y)
        d = descs[i]
        d.type, d.act, d.dX, d.M, d.K = quant.ggml_type, act.to_backend(), x.data_ptr(), M, K.value
        d.dW, d.N, d.dBias, d.dY = weights.data_ptr(), N, (None if bias is None else bias.data_ptr()), y.data_ptr()
    if problems:
        _init(problems[0][0].device.index or 0)
        if norm is None:
            _lib.check(L.gq_qdense_f32_batch(len(problems), descs, _stream_ptr(problems[0][0])))
        else:
            d = norm._desc(problems[0][0].shape[-1])
            fn = L.gq_qdense_norm_bf16_batch if problems[0][0].dtype == torch.bfloat16 else L.gq_qdense_norm_f32_batch
            _lib.check(fn(len(problems), descs, ctypes.byref(d), _stream_ptr(problems[0][0])))
    return outs


# ---- between the q / k / v projections and the output projection of a decoder layer: norms and rotation of queries and keys,
# ---- a key / value cache held in 4 bits, attention over it, eviction from it (ml/layers/attention, attention/kvcache, attention/pos)

_HEAD_DIMS = (64, 128, 256)


def _float_type(name: str, t: torch.Tensor) -> int:
    if t.dtype == torch.float32:
        return _lib.F32
    if t.dtype == torch.bfloat16:
        return _lib.BF16
    raise _lib.NotImplementedByBackend(_lib.ERR_NOT_IMPLEMENTED, f"{name}: dtype {t.dtype} is not implemented")


def _head_rows(name: str, t: torch.Tensor, heads: int | None = None, dim: int | None = None):
    """[rows, heads, dim] with the values of a head side by side; rows and heads may be strided (views of a wider projection)."""
    if not t.is_cuda:
        raise ValueError(f"{name} must be a GPU tensor: this backend has no CPU path")
    if t.dim() != 3 or (heads is not None and t.shape[1] != heads) or (dim is not None and t.shape[2] != dim):
        raise ValueError(f"{name} must be [rows, {'heads' if heads is None else heads}, {'head_dim' if dim is None else dim}], got {tuple(t.shape)}")
    if t.shape[2] > 1 and t.stride(2) != 1:
        raise ValueError(f"{name}: the values of a head must lie side by side")
    return _lib.HeadRowsDesc(t.data_ptr(), t.stride(0), t.stride(1))


def _int32(name: str, t: torch.Tensor, shape: tuple) -> None:
    _require_cuda(name, t)
    if t.dtype != torch.int32 or tuple(t.shape) != shape:
        raise ValueError(f"{name} must be an int32 tensor of shape {shape}, got {t.dtype} {tuple(t.shape)}")


def _kv_desc(cache, page_table, lengths, starts=None, max_new=1, rows=None, accounts=None):
    """gq_kv_cache and the checks that need no look at the device."""
    _require_cuda("cache", cache)
    if cache.dtype != torch.uint8 or cache.dim() != 4 or cache.shape[3] not in tuple(36 * d for d in _HEAD_DIMS):
        raise ValueError("cache must be a Uint8 [pages, kv_heads, page_tokens / 32, 36 * head_dim] tensor (nn.kv_cache)")
    pages, kv_heads, tiles, tile_bytes = cache.shape
    if kv_heads < 1 or tiles < 1:
        raise ValueError(f"cache of shape {tuple(cache.shape)} has no heads or no tokens")
    if lengths.dim() != 1:
        raise ValueError("lengths must be an int32 [sequences] tensor")
    seqs = lengths.shape[0]
    _int32("lengths", lengths, (seqs,))
    if not page_table.is_cuda or page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.shape[0] != seqs or (page_table.shape[1] > 1 and page_table.stride(1) != 1):
        raise ValueError(f"page_table must be an int32 [{seqs}, pages of a sequence] GPU tensor with neighbouring columns side by side")
    if starts is None:
        if rows is not None and rows != seqs:
            raise ValueError(f"without starts every sequence has one row: got {rows} rows for {seqs} sequences")
        if max_new != 1:
            raise ValueError("max_new goes with starts")
        rows = seqs
    else:
        _int32("starts", starts, (seqs + 1,))
        if rows is None:
            raise ValueError("rows must be given with starts")
    if max_new < 1:
        raise ValueError(f"max_new must be at least 1, got {max_new}")
    if accounts is not None:
        _require_cuda("weights", accounts)
        if accounts.dtype != torch.float32 or tuple(accounts.shape) != (pages, kv_heads, 32 * tiles):
            raise ValueError(f"weights must be a float32 [{pages}, {kv_heads}, {32 * tiles}] tensor, got {accounts.dtype} {tuple(accounts.shape)}")
    for name, t in (("page_table", page_table), ("lengths", lengths), ("starts", starts), ("weights", accounts)):
        if t is not None and t.device != cache.device:
            raise ValueError(f"{name} is on {t.device}, the cache on {cache.device}")
    return _lib.KvCacheDesc(cache.data_ptr(), pages, kv_heads, tile_bytes // 36, 32 * tiles, page_table.shape[1], page_table.data_ptr(),
                            max(page_table.stride(0), page_table.shape[1]) if seqs < 2 else page_table.stride(0), lengths.data_ptr(),
                            None if starts is None else starts.data_ptr(), seqs, rows, max_new)


def rotary_table(positions: int, dim: int, base: float = 10000.0, device="cuda") -> tuple:
    """(cos, sin) float32 [positions, dim / 2] for ``qk_norm_rope``: angles position * base^(-2 i / dim), formed in 64 bits.  A model
    with other rates (scaled for long contexts, say) makes its own pair."""
    if dim < 2 or dim % 2:
        raise ValueError(f"dim must be a positive even number, got {dim}")
    rates = base ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    angles = torch.arange(positions, dtype=torch.float64)[:, None] * rates
    return angles.cos().float().to(device), angles.sin().float().to(device)


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, q_norm: RMSNorm | None = None,
                 k_norm: RMSNorm | None = None, interleaved: bool = False, dtype: torch.dtype | None = None) -> tuple:
    """Norms of queries and keys for each head with the rotation by position in the same pass.

    q: [rows, heads, head_dim], k: [rows, key heads, head_dim], float32 or bfloat16, both of one type; rows and heads may be strided.
    positions: int32 [rows]; cos, sin: float32 [table rows, rot / 2] (``rotary_table``).  Values i and i + rot / 2 of a head form a
    pair (``interleaved``: 2 i and 2 i + 1); those from rot on are not rotated.  ``q_norm`` / ``k_norm`` normalise every head over its
    head_dim values first (gain [head_dim]).  Returns (q, k), contiguous, of ``dtype`` (default: the inputs').  A position outside the
    table makes its row NaN."""
    if _lib.fast is not None and (out := _lib.fast.qk_norm_rope(q, k, positions, cos, sin, q_norm, k_norm, interleaved, dtype)) is not None:
        return out
    import ctypes
    xd = _float_type("qk_norm_rope", q)
    if k.dtype != q.dtype:
        raise ValueError(f"q and k differ in type: {q.dtype} vs {k.dtype}")
    dq = _head_rows("q", q)
    rows, heads, dim = q.shape
    dk = _head_rows("k", k, dim=dim)
    if k.shape[0] != rows:
        raise ValueError(f"q and k differ in rows: {rows} vs {k.shape[0]}")
    if dim not in _HEAD_DIMS:
        raise _lib.NotImplementedByBackend(_lib.ERR_NOT_IMPLEMENTED, f"qk_norm_rope: head_dim {dim} is not implemented (64, 128, 256)")
    _int32("positions", positions, (rows,))
    for name, t in (("cos", cos), ("sin", sin)):
        _require_cuda(name, t)
        if t.dtype != torch.float32 or t.dim() != 2 or t.shape != cos.shape:
            raise ValueError(f"{name} must be a float32 [table rows, rot / 2] tensor, cos and sin of one shape")
    for name, t in (("k", k), ("positions", positions), ("cos", cos), ("sin", sin)):
        if t.device != q.device:
            raise ValueError(f"{name} is on {t.device}, q on {q.device}")
    dtype = q.dtype if dtype is None else dtype
    if dtype not in (torch.float32, torch.bfloat16):
        raise _lib.NotImplementedByBackend(_lib.ERR_NOT_IMPLEMENTED, f"qk_norm_rope: output dtype {dtype} is not implemented")
    norms = [None if n is None else n._desc(dim) for n in (q_norm, k_norm)]
    _init(q.device.index or 0)
    q_out = torch.empty(q.shape, dtype=dtype, device=q.device)
    k_out = torch.empty(k.shape, dtype=dtype, device=q.device)
    _lib.check(_lib.lib().gq_qk_norm_rope(xd, ctypes.byref(dq), heads, ctypes.byref(dk), k.shape[1], dim, rows, positions.data_ptr(), cos.data_ptr(), sin.data_ptr(),
                                          cos.shape[0], 2 * cos.shape[1], int(interleaved), *(None if n is None else ctypes.byref(n) for n in norms),
                                          _lib.F32 if dtype == torch.float32 else _lib.BF16, q_out.data_ptr(), k_out.data_ptr(), _stream_ptr(q)))
    return q_out, k_out


def kv_cache(pages: int, kv_heads: int, head_dim: int, page_tokens: int = 64, device="cuda") -> torch.Tensor:
    """An empty key / value cache: uint8 [pages, kv_heads, page_tokens / 32, 36 * head_dim], 4.5 bits a value.

    Groups of 32 neighbouring values of a head share a scale d and stand for d (c - 8) with 4-bit codes c; every value it can hold is
    a float16 number.  A page holds ``page_tokens`` tokens (a multiple of 32) of every key head; which pages a sequence has, and in which
    order, is the caller's table: int32 [sequences, pages of a sequence], where the entries of pages that a sequence does not have (yet)
    may hold anything.  The calls below take it with ``lengths``, int32 [sequences], the tokens of each sequence with the call's new ones.
    A call's rows are one new token per sequence, or, with ``starts`` (int32 [sequences + 1]), rows ``starts[b]`` to ``starts[b + 1]`` the
    new tokens of sequence b, at most ``max_new``: in either case the last tokens of the sequence.  Table, lengths and starts are read
    on the device; a token that the table has no page for is absent: not written, not attended to.  A table may be a slice of the first columns of a wider one: its width bounds the work that is laid out."""
    if head_dim not in _HEAD_DIMS:
        raise _lib.NotImplementedByBackend(_lib.ERR_NOT_IMPLEMENTED, f"kv_cache: head_dim {head_dim} is not implemented (64, 128, 256)")
    if pages < 0 or kv_heads < 1 or page_tokens < 1 or page_tokens % 32:
        raise ValueError(f"kv_cache: {pages} pages, {kv_heads} heads, {page_tokens} tokens a page (a multiple of 32)")
    return torch.zeros((pages, kv_heads, page_tokens // 32, 36 * head_dim), dtype=torch.uint8, device=device)


def kv_cache_append(cache: torch.Tensor, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor,
                    starts: torch.Tensor | None = None, max_new: int = 1, weights: torch.Tensor | None = None) -> None:
    """Writes keys and values [rows, kv_heads, head_dim] (float32 or bfloat16, strided rows and heads allowed) of the new tokens into the cache.

    The scale of a group is minus an eighth of its value of largest magnitude, rounded to 8 significant bits; codes are rounded to
    nearest.  A token with a NaN, an infinity or a magnitude of 65408 or more in a head makes rows that attend to it NaN there.
    ``weights``: the accounts of ``cached_attention``, set to zero for the new tokens."""
    if _lib.fast is not None and _lib.fast.kv_append(cache, k, v, page_table, lengths, starts, max_new, weights):
        return
    import ctypes
    xd = _float_type("kv_cache_append", k)
    if v.dtype != k.dtype or v.shape != k.shape:
        raise ValueError(f"k and v differ: {k.dtype} {tuple(k.shape)} vs {v.dtype} {tuple(v.shape)}")
    d = _kv_desc(cache, page_table, lengths, starts, max_new, k.shape[0] if k.dim() else None, weights)
    dk, dv = (_head_rows(name, t, d.kv_heads, d.head_dim) for name, t in (("k", k), ("v", v)))
    if k.device != cache.device or v.device != cache.device:
        raise ValueError("k, v and the cache must be on one device")
    _init(cache.device.index or 0)
    _lib.check(_lib.lib().gq_kv_append(ctypes.byref(d), xd, ctypes.byref(dk), ctypes.byref(dv), None if weights is None else weights.data_ptr(), _stream_ptr(cache)))


def kv_cache_read(cache: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, starts: torch.Tensor | None = None, max_new: int = 1,
                  rows: int | None = None) -> tuple:
    """(keys, values) float16 [rows, kv_heads, head_dim] that the cache stands for at the last tokens of every sequence, exact.  Rows in
    front of a sequence's first token and rows of absent tokens are zero; rows that belong to no sequence hold anything."""
    if _lib.fast is not None and (out := _lib.fast.kv_read(cache, page_table, lengths, starts, max_new, rows)) is not None:
        return out
    import ctypes
    d = _kv_desc(cache, page_table, lengths, starts, max_new, rows)
    _init(cache.device.index or 0)
    k, v = (torch.empty((d.rows, d.kv_heads, d.head_dim), dtype=torch.float16, device=cache.device) for _ in range(2))
    _lib.check(_lib.lib().gq_kv_read(ctypes.byref(d), k.data_ptr(), v.data_ptr(), _stream_ptr(cache)))
    return k, v


def cached_attention(q: torch.Tensor, cache: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, starts: torch.Tensor | None = None,
                     max_new: int = 1, scale: float | None = None, window: int = 0, weights: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(scale q . k) v of the new tokens over a 4-bit cache (which already holds them).

    q: [rows, heads, head_dim] float32 or bfloat16, strided rows and heads allowed; ``heads`` is a multiple of the cache's key heads and
    neighbouring query heads share one.  ``scale`` defaults to head_dim^-1/2.  A token sees itself and the tokens in front of it in its
    sequence, with a ``window`` the last that many; one that sees nothing gets zeros.  ``weights``: float32 [pages, kv_heads, page_tokens],
    to which the softmax weights that every cached token receives are added (summed over rows and the query heads of a key head): what
    ``kv_cache_evict`` goes by.  Sequences may share pages (a common beginning, say), with ``weights`` they must not.  Every row of q belongs to a
    sequence.  Returns [rows, heads, head_dim] of q's type, contiguous."""
    if _lib.fast is not None and (out := _lib.fast.cached_attention(q, cache, page_table, lengths, starts, max_new, scale, window, weights)) is not None:
        return out
    import ctypes
    xd = _float_type("cached_attention", q)
    d = _kv_desc(cache, page_table, lengths, starts, max_new, q.shape[0] if q.dim() else None, weights)
    dq = _head_rows("q", q, dim=d.head_dim)
    heads = q.shape[1]
    if heads < 1 or heads % d.kv_heads:
        raise ValueError(f"{heads} query heads are not a multiple of {d.kv_heads} key heads")
    if window < 0:
        raise ValueError(f"window must not be negative, got {window}")
    if q.device != cache.device:
        raise ValueError("q and the cache must be on one device")
    _init(cache.device.index or 0)
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    _lib.check(_lib.lib().gq_kv_attention(ctypes.byref(d), xd, ctypes.byref(dq), heads, d.head_dim ** -0.5 if scale is None else scale, window,
                                          None if weights is None else weights.data_ptr(), out.data_ptr(), _stream_ptr(cache)))
    return out


def kv_cache_evict(cache: torch.Tensor, weights: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, keep: int, recent: int = 0) -> tuple:
    """Shrinks every sequence of more than ``keep`` tokens to ``keep``: for each key head the last ``recent`` tokens and the keep - recent
    others of largest accumulated weight stay (ties: the earlier token), moved to the front of the sequence's pages in their order,
    with their weights.  Returns (kept, lengths): int32 [sequences, kv_heads, keep] former places of the kept tokens (-1 behind the last), and
    the new lengths, min(length, keep); ``lengths`` itself is left as it is.  Sequences must not share pages."""
    if _lib.fast is not None and (out := _lib.fast.kv_evict(cache, weights, page_table, lengths, keep, recent)) is not None:
        return out
    import ctypes
    d = _kv_desc(cache, page_table, lengths, accounts=weights)
    if weights is None:
        raise ValueError("weights must not be None")
    if keep < 1 or not 0 <= recent <= keep:
        raise ValueError(f"keep must be positive and recent between 0 and keep: got {keep}, {recent}")
    _init(cache.device.index or 0)
    kept = torch.empty((d.seqs, d.kv_heads, keep), dtype=torch.int32, device=cache.device)
    new_lengths = torch.empty_like(lengths)
    _lib.check(_lib.lib().gq_kv_evict(ctypes.byref(d), weights.data_ptr(), keep, recent, kept.data_ptr(), new_lengths.data_ptr(), _stream_ptr(cache)))
    return kept, new_lengths
