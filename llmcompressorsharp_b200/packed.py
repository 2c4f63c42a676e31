"""Packed 4-bit weights that a compressed model runs from, and the embedding.

The modifiers leave 4-bit codes with scales and zero-points in ``state.compressed``
(GPTQModifier.cs:108-137, RtnModifier.cs:44-122); the reference only dequantises such codes
(Int4PackedTensor.cs:152-161).  Here

- ``Int4Weight`` lays one weight's codes out once for the kernels;
- ``int4_linear`` multiplies by it, one token or many, with the gradients of x and the bias;
- ``embedding`` looks tokens up in a dense or packed table, with the gradient of a dense one;
- ``Int4Linear`` / ``Int4Embedding`` are the modules, and ``load_compressed`` puts them into a
  model in place of the ``torch.nn.Linear`` / ``Embedding`` modules whose weights were compressed.

Results are new tensors on the current stream of their device; scratch comes from torch's
allocator, so calls can be captured into CUDA graphs and run on several streams at once.
"""

from __future__ import annotations

import ctypes as C

import torch
import torch.autograd.forward_ad as forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from ._device import target_device, to_device
from .errors import ArgumentError, InvalidOperationError, NotSupportedError, ShapeError

_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}


def _dtype(t: torch.Tensor, name: str) -> int:
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise ArgumentError(f"{name} must be float32, bfloat16 or float16 (got {t.dtype})")
    return code


def _rows(t: torch.Tensor, last: int) -> torch.Tensor:
    """t as [rows, last] whose rows are contiguous and do not overlap."""
    if t.dim() != 2:
        t = t.reshape(-1, last)
    if t.stride(1) != 1 and last != 1 or t.stride(0) < last and t.shape[0] > 1:
        t = t.contiguous()
    return t


def _pitch(t: torch.Tensor) -> int:
    """Elements between rows (of at most one row: its length, whatever stride torch keeps)."""
    return t.stride(0) if t.shape[0] > 1 else max(1, t.shape[1])


_is_tracing, _transform, _modes = torch._C._is_tracing, torch._C._functorch.peek_interpreter_stack, torch._C._len_torch_dispatch_stack


def _refuse_unseen(name: str, a, b):
    """Refuses a call whose operators torch watches: a trace of the library's calls would hold empty tensors in place of
    their results, a transform would lose its part of them.  (0.3 us where nothing does.)"""
    if not (_is_tracing() or _modes()) and _transform() is None and type(a) in _PLAIN and type(b) in _PLAIN:
        return
    tensors = [t for t in (a, b) if isinstance(t, torch.Tensor)]
    what = None
    if _is_tracing():
        what = "torch.jit's tracing"
    elif any(torch._C._functorch.is_functorch_wrapped_tensor(t) for t in tensors):
        what = "a torch.func transform"
    elif _modes() and torch._C._get_dispatch_mode(torch._C._TorchDispatchModeKey.PROXY) is not None:
        what = "torch.fx's tracing"
    else:
        from torch._subclasses import FakeTensor

        if any(isinstance(t, FakeTensor) for t in tensors):
            what = "a FakeTensor"
    if what is not None:
        raise NotSupportedError(f"{name} cannot run under {what}: its kernels are not torch operators")


class Int4Weight:
    """A [rows, cols] weight of 4-bit codes: W[n][k] = (q - zp) * s, one (s, zp) per ``group_size``
    columns of a row (strategy "group"), per row ("channel") or for all of it ("tensor").

    ``codes`` are as ``rtn_quantize`` and the GPTQ calls write them for num_bits <= 4:
    (q - zp) & 0xF, two per byte, the even column in the high nibble (Int4PackedTensor.cs:47-69).
    They are laid out anew (and rounded up to 128 rows and columns); the tensors passed in are not
    kept.  Zero-points are in [0, 2^num_bits).  Groups have at least 16 columns.  The weight is constant: its scales take no gradient.  It
    stays on its device (a module's ``to`` does not move it) and is in no ``state_dict``; it can be
    copied and pickled."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, zero_points: torch.Tensor | None, cols: int,
                 strategy: str = "group", group_size: int = 128, symmetric: bool = True, num_bits: int = 4):
        if codes is None or scales is None:
            raise ArgumentError("codes and scales must not be null")
        if num_bits not in (2, 3, 4):
            raise NotSupportedError(f"a packed 4-bit weight takes codes of 2 to 4 bits (got {num_bits})")
        if strategy not in ("tensor", "channel", "group"):
            raise NotSupportedError(f"a packed 4-bit weight has a tensor, channel or group strategy (got {strategy})")
        if not symmetric and zero_points is None:
            raise ArgumentError("an asymmetric grid needs zero-points")
        if codes.dim() != 2 or codes.dtype != torch.uint8 or codes.shape[1] != (cols + 1) // 2:
            raise ShapeError(f"codes must be uint8 [rows, {(cols + 1) // 2}] for {cols} columns "
                             f"(got {codes.dtype} {list(codes.shape)})")
        if scales.requires_grad:
            raise InvalidOperationError("a packed weight's scales take no gradient")
        rows = codes.shape[0]
        group = int(group_size) if strategy == "group" else max(1, int(cols))
        size, exps = _lib.I64(), _lib.I64()
        _lib.call("llmc_int4_layout_sizes", rows, cols, group, C.byref(size), C.byref(exps))
        want = {"tensor": 1, "channel": rows, "group": rows * -(-cols // group)}[strategy]
        for name, t in (("scales", scales), ("zero_points", zero_points)):
            if t is not None and t.numel() != want:
                raise ShapeError(f"{name} must have {want} entries for strategy {strategy} (got {t.numel()})")
        dev = target_device(codes, scales)
        self.device = torch.device("cuda", dev.index if dev.index is not None else torch.cuda.current_device())
        self.shape = (rows, int(cols))
        self.strategy, self.symmetric, self.num_bits = strategy, bool(symmetric), int(num_bits)
        self.group_size = group
        c = to_device(codes.detach(), self.device)
        s = to_device(scales.detach(), self.device, torch.float32)
        z = to_device(zero_points.detach(), self.device, torch.int32) if not symmetric else None
        self.packed = torch.empty(size.value, dtype=torch.uint8, device=self.device)
        self.exps = torch.empty(exps.value, dtype=torch.int32, device=self.device)
        self._bind()
        _lib.call("llmc_int4_layout", self._ctx, _lib.stream(self._index), _lib.ptr(c), c.shape[1], _lib.ptr(s), _lib.ptr(z),
                  _lib.STRATEGY[strategy], int(symmetric), self._ref)

    def _bind(self):
        self._c = _lib.Int4WeightC(self.packed.data_ptr(), self.exps.data_ptr(), *self.shape, self.group_size)
        self._ref = C.byref(self._c)
        self._ctx, self._index = _lib.ctx_handle(self.device.index), self.device.index
        self._need: dict = {}

    def __getstate__(self):
        return {k: v for k, v in self.__dict__.items() if k not in ("_c", "_ref", "_ctx", "_index", "_need")}

    def __setstate__(self, state):
        self.__dict__.update(state)
        self.device = self.packed.device
        self._bind()

    @staticmethod
    def from_entry(entry: dict, cols: int) -> "Int4Weight":
        """From one weight's entry of ``state.compressed`` (or ``CompressedTensorsWriter.entries_from_pipeline``)."""
        if entry is None or entry.get("codes") is None:
            raise ArgumentError("the entry has no codes")
        return Int4Weight(entry["codes"], entry["scales"], entry["zero_points"], cols, entry["strategy"],
                          entry["group_size"], entry["symmetric"], entry["num_bits"])

    @staticmethod
    def from_float(weight: torch.Tensor, config) -> "Int4Weight":
        """Round-to-nearest of a dense [rows, cols] weight with an ``RtnConfig`` of at most 4 bits."""
        from .rtn import rtn_quantize

        if weight is None or weight.dim() != 2:
            raise ArgumentError("weight must be a matrix")
        if config.num_bits > 4:
            raise NotSupportedError(f"a packed 4-bit weight takes codes of 2 to 4 bits (got {config.num_bits})")
        _, codes, scales, zps = rtn_quantize(weight, config, want_codes=True, want_deq=False)
        return Int4Weight(codes, scales, zps, weight.shape[1], config.strategy, config.group_size, config.symmetric,
                          config.num_bits)

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """[rows, cols] of (q - zp) * s, rounded once to ``dtype``."""
        if dtype not in _DTYPES:
            raise ArgumentError(f"dtype must be float32, bfloat16 or float16 (got {dtype})")
        out = torch.empty(self.shape, dtype=dtype, device=self.device)
        _lib.call("llmc_int4_dequantize", self._ctx, _lib.stream(self._index), self._ref, _DTYPES[dtype], out.data_ptr(),
                  self.shape[1])
        return out

    def _workspace(self, fn: str, at: int, code: int, tokens: int, ld: int):
        """Scratch tensor (or None) of one product of the rows at address ``at``; its size depends on what the key holds."""
        key = (fn, code, tokens, ld, at % 16)
        need = self._need.get(key)
        if need is None:
            v = _lib.I64()
            _lib.call(fn, self._ctx, self._ref, at, code, tokens, ld, C.byref(v))
            if len(self._need) >= 256:
                self._need.clear()
            need = self._need[key] = v.value
        return torch.empty(need, dtype=torch.uint8, device=self.device) if need else None

    def _product(self, x: torch.Tensor, bias, back: bool) -> torch.Tensor:
        """x [..., cols] W^T + bias, or (back) x [..., rows] W; a new tensor [..., rows] or [..., cols]."""
        last = self.shape[0 if back else 1]
        if x.is_contiguous():
            a, tokens, ld = x, x.numel() // last, last
        else:
            a = _rows(x, last)
            tokens, ld = a.shape[0], _pitch(a)
        n = self.shape[1 if back else 0]
        out = x.new_empty(*x.shape[:-1], n)
        if tokens == 0:
            return out
        code, at = _DTYPES[a.dtype], a.data_ptr()
        ws = self._workspace("llmc_int4_linear_grad_workspace" if back else "llmc_int4_linear_workspace", at, code, tokens, ld)
        wp, wn = (ws.data_ptr(), ws.numel()) if ws is not None else (None, 0)
        if back:
            _lib.call("llmc_int4_linear_grad", self._ctx, _lib.stream(self._index), self._ref, at, code, tokens, ld, out.data_ptr(), n, wp, wn)
        else:
            _lib.call("llmc_int4_linear", self._ctx, _lib.stream(self._index), self._ref, at, code, tokens, ld,
                      bias.data_ptr() if bias is not None else None, out.data_ptr(), n, wp, wn)
        return out


# What the calls get outside torch's transforms and traces; they look closer at anything else.
_PLAIN = frozenset((torch.Tensor, torch.nn.Parameter, Int4Weight, type(None)))
_needs: dict = {}  # (call, device, sizes) -> bytes of scratch


def _scratch(fn: str, index: int, device, *sizes) -> torch.Tensor:
    """Scratch tensor of a call whose need depends on its sizes alone."""
    key = (fn, index, sizes)
    need = _needs.get(key)
    if need is None:
        v = _lib.I64()
        _lib.call(fn, _lib.ctx_handle(index), *sizes, C.byref(v))
        if len(_needs) >= 256:
            _needs.clear()
        need = _needs[key] = v.value
    return torch.empty(need, dtype=torch.uint8, device=device)


def _col_sum(x2: torch.Tensor) -> torch.Tensor:
    index = x2.device.index
    ctx = _lib.ctx_handle(index)
    rows, cols = x2.shape
    ws = _scratch("llmc_col_sum_workspace", index, x2.device, rows, cols)
    out = torch.empty(cols, dtype=x2.dtype, device=x2.device)
    _lib.call("llmc_col_sum", ctx, _lib.stream(index), x2.data_ptr(), _DTYPES[x2.dtype], rows, cols, _pitch(x2), out.data_ptr(),
              ws.data_ptr(), ws.numel())
    return out


def _once(backward):
    """once_differentiable, whose wrapping a pass that records no graph goes without."""
    guarded = once_differentiable(backward)
    return lambda ctx_, dy: guarded(ctx_, dy) if torch.is_grad_enabled() else backward(ctx_, dy)


def _linear_in(f, dy):
    """f(dy) of a linear f, with its tangent where dy has one (forward mode over a backward pass)."""
    if forward_ad._current_level < 0:
        return f(dy)
    dy, tangent = forward_ad.unpack_dual(dy)
    return f(dy) if tangent is None else forward_ad.make_dual(f(dy), f(tangent))


class _Int4LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx_, x, weight, bias):
        ctx_.weight = weight
        return weight._product(x, bias, False)

    @staticmethod
    @_once
    def backward(ctx_, dy):
        w = ctx_.weight
        dx = _linear_in(lambda d: w._product(d, None, True), dy) if ctx_.needs_input_grad[0] else None
        db = _linear_in(lambda d: _col_sum(_rows(d, w.shape[0])), dy) if ctx_.needs_input_grad[2] else None
        return dx, None, db


def int4_linear(x: torch.Tensor, weight: Int4Weight, bias: torch.Tensor | None = None) -> torch.Tensor:
    """y = x W^T + bias for x [..., cols] of float32, bfloat16 or float16; y [..., rows] of x's type.

    Sums are fp32 and rounded once.  With few rows of x (32 and fewer always, up to 256 in many cases) the
    codes are multiplied as exact integers; with more, and in the backward pass, W is rounded to x's 16-bit
    type first (as a dequantised weight of that type is), or for float32 each product is kept to 2^-22 of itself.
    In float16 a scale below 2^-13 of the largest in its row (in the backward pass: of its group's in any row) loses bits
    then.  Differentiable once,
    in x and the bias, backward or forward (``torch.autograd.forward_ad``); not under ``torch.func`` or a trace."""
    if x is None or weight is None:
        raise ArgumentError("x and weight must not be null")
    if not isinstance(weight, Int4Weight):
        raise ArgumentError(f"weight must be an Int4Weight (got {type(weight).__name__})")
    _refuse_unseen("int4_linear", x, bias)
    _dtype(x, "x")
    rows, cols = weight.shape
    if x.dim() == 0 or x.shape[-1] != cols:
        raise ShapeError(f"Input last dim ({x.shape[-1] if x.dim() else 'scalar'}) must equal the weight's columns ({cols}).")
    if x.device != weight.device:
        raise ArgumentError(f"x is on {x.device}, the weight on {weight.device}")
    if bias is not None:
        if bias.dim() != 1 or bias.shape[0] != rows:
            raise ShapeError(f"bias must have {rows} entries (got {list(bias.shape)})")
        if bias.dtype != x.dtype or bias.device != x.device:
            raise ArgumentError(f"bias must be {x.dtype} on {x.device} (got {bias.dtype} on {bias.device})")
        if bias.stride(0) != 1:
            bias = bias.contiguous()
    if forward_ad._current_level >= 0:
        (x, dx), (bias, db) = forward_ad.unpack_dual(x), (None, None) if bias is None else forward_ad.unpack_dual(bias)
        if dx is not None or db is not None:
            y = _linear(x, weight, bias)
            dy = db.expand_as(y).contiguous() if dx is None else _linear(dx, weight, None if db is None else db.contiguous())
            return forward_ad.make_dual(y, dy)
    return _linear(x, weight, bias)


def _linear(x, weight, bias):
    if torch.is_grad_enabled() and (x.requires_grad or (bias is not None and bias.requires_grad)):
        return _Int4LinearFn.apply(x, weight, bias)
    return weight._product(x, bias, False)


def _lookup(ids, table, scale):
    out = table.new_empty(*ids.shape, table.shape[1])
    index = table.device.index
    _lib.call("llmc_embedding", _lib.ctx_handle(index), _lib.stream(index), ids.data_ptr(), int(ids.dtype == torch.int64),
              ids.numel(), table.data_ptr(), _DTYPES[table.dtype], table.shape[0], table.shape[1], _pitch(table), scale,
              out.data_ptr(), table.shape[1])
    return out


def _table_grad(ids, dy, shape, scale, padding):
    vocab, hidden = shape
    d2 = _rows(dy, hidden)
    index = dy.device.index
    ctx = _lib.ctx_handle(index)
    ws = _scratch("llmc_embedding_grad_workspace", index, dy.device, ids.numel(), vocab, hidden)
    out = torch.empty(vocab, hidden, dtype=dy.dtype, device=dy.device)
    _lib.call("llmc_embedding_grad", ctx, _lib.stream(index), ids.data_ptr(), int(ids.dtype == torch.int64), ids.numel(),
              d2.data_ptr(), _DTYPES[dy.dtype], _pitch(d2), vocab, hidden, scale, padding, out.data_ptr(), ws.data_ptr(), ws.numel())
    return out


class _EmbeddingFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx_, table, ids, scale, padding):
        ctx_.save_for_backward(ids)
        ctx_.scale, ctx_.padding, ctx_.shape = scale, padding, table.shape
        return _lookup(ids, table, scale)

    @staticmethod
    @_once
    def backward(ctx_, dy):
        (ids,) = ctx_.saved_tensors
        return _linear_in(lambda d: _table_grad(ids, d, ctx_.shape, ctx_.scale, ctx_.padding), dy), None, None, None


def embedding(ids: torch.Tensor, table, scale: float = 1.0, padding_idx: int | None = None,
              dtype: torch.dtype | None = None) -> torch.Tensor:
    """scale * table[ids], rounded once: ids [...] int64 or int32, table [vocab, hidden] dense or an
    ``Int4Weight``; the result is [..., hidden] of the dense table's type, or of ``dtype`` (default
    bfloat16) for a packed one.

    Differentiable in a dense table: row v gets scale times the sum of dy over its tokens, added in fp32 in a fixed
    order (by token; of more than 32, runs of 32 tokens and then their sums; the same bits every time), the row ``padding_idx`` zeros; once, or forward
    (``torch.autograd.forward_ad``); not under ``torch.func`` or a trace.  An id outside the table gives
    a row of zeros and no gradient, and the device's next ``llmc_sync`` raises ArgumentOutOfRangeError."""
    if ids is None or table is None:
        raise ArgumentError("ids and table must not be null")
    if ids.dtype not in (torch.int64, torch.int32):
        raise ArgumentError(f"ids must be int64 or int32 (got {ids.dtype})")
    packed = isinstance(table, Int4Weight)
    _refuse_unseen("embedding", ids, table)
    if not packed:
        if table.dim() != 2:
            raise ShapeError(f"table must be [vocab, hidden] (got {list(table.shape)})")
        _dtype(table, "table")
        if dtype is not None and dtype != table.dtype:
            raise ArgumentError(f"a dense table is looked up in its own type ({table.dtype}, asked for {dtype})")
        if not table.is_cuda:
            raise ArgumentError(f"the table must be on a CUDA device (got {table.device})")
        if 0 in table.shape:
            raise ShapeError(f"a table needs positive sizes (got {list(table.shape)})")
    if ids.device != table.device:
        raise ArgumentError(f"ids are on {ids.device}, the table on {table.device}")
    vocab, hidden = table.shape
    padding = -1 if padding_idx is None else int(padding_idx)
    if padding_idx is not None:
        if not -vocab <= padding < vocab:
            raise ArgumentError(f"padding_idx {padding_idx} is outside the table of {vocab} rows")
        padding %= vocab
    ids = ids.contiguous()
    scale = float(scale)
    if packed:
        dtype = dtype or torch.bfloat16
        if dtype not in _DTYPES:
            raise ArgumentError(f"dtype must be float32, bfloat16 or float16 (got {dtype})")
        out = torch.empty(*ids.shape, hidden, dtype=dtype, device=table.device)
        _lib.call("llmc_int4_embedding", table._ctx, _lib.stream(table._index), ids.data_ptr(), int(ids.dtype == torch.int64),
                  ids.numel(), table._ref, _DTYPES[dtype], scale, out.data_ptr(), hidden)
        return out
    if forward_ad._current_level >= 0:
        table, tangent = forward_ad.unpack_dual(table)
        if tangent is not None:
            return forward_ad.make_dual(_dense_embedding(ids, table, scale, padding), _dense_embedding(ids, tangent, scale, padding))
    return _dense_embedding(ids, table, scale, padding)


def _dense_embedding(ids, table, scale, padding):
    table = _rows(table, table.shape[1])
    if torch.is_grad_enabled() and table.requires_grad:
        return _EmbeddingFn.apply(table, ids, scale, padding)
    return _lookup(ids, table, scale)


class Int4Linear(torch.nn.Module):
    """``torch.nn.Linear`` with a packed weight."""

    def __init__(self, weight: Int4Weight, bias: torch.Tensor | None = None):
        super().__init__()
        self.packed_weight = weight
        self.out_features, self.in_features = weight.shape
        if isinstance(bias, torch.nn.Parameter):
            self.bias = bias
        else:
            self.register_buffer("bias", bias)

    def forward(self, x):
        bias = self.bias
        if torch.is_autocast_enabled("cuda") and x.is_cuda and x.dtype in _DTYPES:  # as torch.nn.Linear is cast
            dtype = torch.get_autocast_dtype("cuda")
            x, bias = x.to(dtype), None if bias is None else bias.to(dtype)
        return int4_linear(x, self.packed_weight, bias)

    def extra_repr(self):
        w = self.packed_weight
        return f"in_features={self.in_features}, out_features={self.out_features}, strategy={w.strategy}, group_size={w.group_size}"


class Int4Embedding(torch.nn.Module):
    """``torch.nn.Embedding`` with a packed table, returning ``dtype``."""

    def __init__(self, weight: Int4Weight, dtype: torch.dtype = torch.bfloat16, scale: float = 1.0):
        super().__init__()
        self.packed_weight = weight
        self.num_embeddings, self.embedding_dim = weight.shape
        self.dtype, self.scale = dtype, scale

    def forward(self, ids):
        return embedding(ids, self.packed_weight, self.scale, dtype=self.dtype)


class TokenEmbedding(torch.nn.Embedding):
    """``torch.nn.Embedding`` whose lookup, on a CUDA device, is the library's (the same values; a gradient with the same
    bits every time).  Types and options that it does not take, other devices, and what torch transforms or records
    (forward mode, ``torch.func``, tracing, compiling, dispatch modes, subclasses of Tensor) are torch's.  Two things differ from torch's on a
    device: it is differentiable once, and an id outside the table is no device assertion but a row of zeros, which the
    device's next ``llmc_sync`` reports."""

    def forward(self, ids):
        w = self.weight
        if (w.is_cuda and w.dtype in _DTYPES and ids.dtype in (torch.int64, torch.int32) and type(ids) is torch.Tensor
                and type(w) in (torch.Tensor, torch.nn.Parameter)
                and self.max_norm is None and not self.scale_grad_by_freq and not self.sparse
                and forward_ad._current_level < 0 and not torch.compiler.is_compiling() and not _is_tracing()
                and _transform() is None and not _modes()):
            return embedding(ids, w, padding_idx=self.padding_idx)
        return super().forward(ids)


def check_ids(model: torch.nn.Module) -> None:
    """Waits for the devices of the library's embeddings in ``model`` and raises ArgumentOutOfRangeError if a lookup on one
    of them, since the last check, had an id outside its table (its row was zeros).  Other pending errors of the device
    are raised as well."""
    if model is None:
        raise ArgumentError("model must not be null")
    devices = {m.packed_weight.device if isinstance(m, Int4Embedding) else m.weight.device
               for m in model.modules() if isinstance(m, (Int4Embedding, TokenEmbedding))}
    for device in devices:
        if device.type == "cuda":
            _lib.call("llmc_sync", _lib.ctx_for(device.index))


# What a module holds for its caller around its forward pass.  The dicts are shared, so that a hook's handle still
# takes it out.
_HOOKS = ("_forward_hooks", "_forward_hooks_with_kwargs", "_forward_hooks_always_called", "_forward_pre_hooks",
          "_forward_pre_hooks_with_kwargs", "_backward_hooks", "_backward_pre_hooks", "_is_full_backward_hook")


def load_compressed(model: torch.nn.Module, compressed: dict) -> list[str]:
    """Puts packed modules into ``model`` for the entries of ``state.compressed`` (weight name ->
    entry): a Linear or Embedding whose ``<module>.weight`` has 4-bit codes is replaced, wherever the model holds it,
    by an Int4Linear / Int4Embedding that returns the old weight's type, with its forward and backward hooks and its
    ``training`` flag.  Entries without codes, of more than 4 bits or of other modules stay dense: subclasses too, whose
    forward may compute more, an Embedding with max_norm, and a module whose weight is of another type than float32,
    bfloat16 and float16 or is no parameter of its own (a hook computes it).  So does a module that was tied to a
    replaced one's weight.  Returns the names of the modules replaced.

    A packed weight is on the CUDA device of its codes (the current one for codes on the CPU), whatever the old module's
    device: move the rest of a model on the CPU there.  It takes a quarter of the memory and reads, which decides a
    product of few tokens; one of some thousand tokens takes 1.2 to 1.3 times as long as with the 16-bit weight."""
    if model is None or compressed is None:
        raise ArgumentError("model and compressed must not be null")
    modules, done = dict(model.named_modules(remove_duplicate=False)), []
    for name, entry in compressed.items():
        if not name.endswith(".weight") or entry.get("codes") is None or entry["num_bits"] > 4:
            continue
        path = name[: -len(".weight")]
        old = modules.get(path)
        if not path or type(old) not in (torch.nn.Linear, torch.nn.Embedding, TokenEmbedding):
            continue
        if isinstance(old, torch.nn.Embedding) and old.max_norm is not None:
            continue
        if "weight" not in old._parameters or old.weight.dtype not in _DTYPES:
            continue
        w = Int4Weight.from_entry(entry, old.weight.shape[1])
        if w.shape != tuple(old.weight.shape):
            raise ShapeError(f"{name}: codes are {list(w.shape)}, the module's weight {list(old.weight.shape)}")
        if isinstance(old, torch.nn.Linear):
            new = Int4Linear(w, old.bias)
        else:
            new = Int4Embedding(w, old.weight.dtype)
        for hooks in _HOOKS:
            setattr(new, hooks, getattr(old, hooks))
        new.training = old.training
        for at in [p for p, m in modules.items() if m is old]:
            parent, _, leaf = at.rpartition(".")
            setattr(modules[parent], leaf, new)
            modules[at] = new
        done.append(path)
    return done
