"""A decoder layer's linears in 8 bits on the HIP library: e4m3 rows and weights with a power-of-two scale per block of
128, which the matrix instructions apply themselves.

* ``Weight`` — a linear's weight ``[N, K]`` (or a fused gate/up one) in 8 bits, laid out once in the order the matrix
  instructions read: half the bytes of the 16-bit packed weights, which a round is bound by, and twice the
  matrix rate, which a prompt is bound by;
* ``Rows`` — activations ``[M, K]`` in 8 bits; ``quantize`` makes them, and ``rms_norm`` with ``dtype=float8_e4m3fn``;
* ``linear`` — rows times a weight, transposed: the 8-bit form of ``fast_gemm.hip_linear``;
* ``gate_up_silu`` — the gate/up projection with its activation: that of ``fast_gemm.gate_up_silu``;
* ``rms_norm`` — the root-mean-square norm between them, with the residual's addition, in 8 or 16 bits.

A block's scale is the least power of two s with (largest finite magnitude) <= 448 s, at least 2^-64, as in the paged
cache; codes are rounded to nearest even, and what is not finite becomes NaN, in its own row alone. A row's blocks are 128
of K, a weight's 128 x 128. ``linear`` and ``gate_up_silu`` take 16-bit rows too, which they round as ``quantize`` does.

Calls run on the current stream of the tensors' GPU, allocate what they return, keep nothing between calls and can be
captured; sums are in one order, so results repeat bit for bit. Nothing here has a derivative: tensors that require a
gradient are refused while gradients are recorded, and so are those that carry a forward-mode tangent, and calls while a
tracer records.
"""

from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import _lib

E4M3 = torch.float8_e4m3fn
BLOCK = 128
_CODES = _lib.DTYPE_CODES
_OUT = {torch.bfloat16: _lib.PLM_FP8_BF16, torch.float16: _lib.PLM_FP8_F16, torch.float32: _lib.PLM_FP8_F32}
_EPS = (2.0 ** -100, 2.0 ** 100)
_IN = {_lib.PLM_BF16: _lib.PLM_FP8_ROWS_BF16, _lib.PLM_F16: _lib.PLM_FP8_ROWS_F16}   # plm_fp8_in of a plm_dtype
MOST = 1 << 21   # rows of a product's operands


# What follows is on every call's path, where the host's time counts: one look at each property, strides only of tensors that
# are not contiguous, messages formed for refusals alone, sizes given one by one (a tuple of them costs an allocation 0.2 us more).


def _run(entry, index: int, *args) -> int:
    """Status of a C entry on GPU ``index``, on its current stream."""
    if torch._C._is_tracing():
        raise RuntimeError("a tracer would record the 8-bit calls' allocations and not what fills them: call them outside of it")
    if index == torch._C._cuda_getDevice():
        return entry(*args, torch._C._cuda_getCurrentRawStream(index))
    with torch.cuda.device(index):
        return entry(*args, torch._C._cuda_getCurrentRawStream(index))


def _derivative(t: torch.Tensor, name: str) -> None:
    """Refuses a tensor whose derivative a call would drop."""
    if t.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{name} requires a gradient, and the 8-bit calls have none: detach it, or call under no_grad")
    # Tangents live inside a dual level only; asking for one takes ten times as long as asking for the level.
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        raise RuntimeError(f"{name} carries a forward-mode tangent, and the 8-bit calls have none: detach it")


def _no_memory(name: str) -> None:
    # A stand-in for a tensor (a tracer's, a wrapper's): its null would be taken for an argument that is not given.
    raise RuntimeError(f"{name} has no memory that a kernel could read")


def _matrix(t: torch.Tensor, name: str, index: int | None = None) -> tuple[torch.Tensor, int, int, int, int, int, int]:
    """``t`` [rows, k] of 16 bits as a kernel can read it, its pointer, row stride, type's code, GPU, rows and k."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if t.dim() != 2:
        raise ValueError(f"{name} must be [rows, k], got {list(t.shape)}")
    code = _CODES.get(t.dtype)
    if code is None:
        raise TypeError(f"{name} must be bf16 or fp16, got {t.dtype}")
    if t.requires_grad or forward_ad._current_level >= 0:
        _derivative(t, name)
    rows, k = t.shape
    if k < 8 or k % 8 or k > 1 << 24:
        raise ValueError(f"{name}'s rows must have a multiple of 8 in [8, 2^24] of elements, got {k}")
    on = t.get_device()
    if on < 0 or (index is not None and on != index):
        raise RuntimeError(f"{name} must be on {'a GPU' if index is None else f'cuda:{index}'}, got {t.device}")
    at = t.data_ptr()
    if not at and rows:
        _no_memory(name)
    if at % 16 == 0:
        if t.is_contiguous():
            return t, at, k, code, on, rows, k
        stride, one = t.stride()
        if one == 1 and stride % 8 == 0:
            return t, at, stride, code, on, rows, k
    t = t.clone(memory_format=torch.contiguous_format)
    return t, t.data_ptr(), k, code, on, rows, k


class _Eight:
    """Codes and scales of ``rows`` rows of ``k`` (``include/plm_amd.h`` states their order); what it was made of stays."""

    _gate_up = False

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, rows: int, k: int):
        lib = _lib.lib()
        need = int(lib.plm_fp8_codes_bytes(rows, k)), int(lib.plm_fp8_scales_bytes(rows, k))
        if not need[0]:
            raise ValueError(f"8-bit rows need 1 to 2^24 - 1 rows of a multiple of 8 in [8, 2^24], at most 2^25 fragments, got "
                             f"[{rows}, {k}]")
        for name, t, size, dtype in (("codes", codes, need[0], E4M3), ("scales", scales, need[1], torch.uint8)):
            if t.dtype is not dtype or t.shape != (size,) or not t.is_contiguous() or t.data_ptr() % 16:
                raise ValueError(f"{name} of [{rows}, {k}] must be contiguous {dtype} [{size}] on 16 bytes, got {t.dtype} "
                                 f"{list(t.shape)}")
        _derivative(codes, "codes")
        if not codes.is_cuda or scales.device != codes.device:
            raise RuntimeError(f"codes and scales live on one GPU; got {codes.device} and {scales.device}")
        self.__dict__.update(codes=codes, scales=scales, rows=rows, k=k, _index=codes.get_device(), codes_at=codes.data_ptr(),
                             scales_at=scales.data_ptr())

    @classmethod
    def _new(cls, rows: int, k: int, like: torch.Tensor):
        """Uninitialised rows on ``like``'s GPU, for a kernel to fill: one allocation, no check of what is known."""
        frags, blocks = (rows + 15) // 16, (k + 127) // 128
        codes = frags * blocks * 2048
        both = like.new_empty(codes + frags * ((blocks + 3) // 4) * 64, dtype=torch.uint8)
        self = cls.__new__(cls)
        at = both.data_ptr()
        d = self.__dict__
        d["_both"], d["rows"], d["k"], d["_index"], d["codes_at"], d["scales_at"] = both, rows, k, like.get_device(), at, at + codes
        return self

    def __getattr__(self, name: str):
        # The tensors of what a kernel filled, as views when they are asked for.
        if name in ("codes", "scales") and "_both" in self.__dict__:
            both, size = self._both, self.scales_at - self.codes_at
            return both[:size].view(E4M3) if name == "codes" else both[size:]
        raise AttributeError(name)

    def __reduce__(self):
        # A copy's addresses are its own tensors'; bytes, as pickle knows no float8.
        return _again, (type(self), self.codes.view(torch.uint8), self.scales, self.rows, self.k, self._gate_up)

    @property
    def device(self) -> torch.device:
        return torch.device("cuda", self._index)

    def __setattr__(self, name: str, value) -> None:
        raise AttributeError(f"8-bit rows stay what they were made of: {name} cannot be set")

    def __delattr__(self, name: str) -> None:
        raise AttributeError(f"8-bit rows keep their {name}")

    @property
    def shape(self) -> tuple[int, int]:
        return self.rows, self.k

    def values(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """``[rows, k]``: what the codes stand for, exact in bf16 and fp32 but for codes that round up to 2^128,
        which are infinite (fp16 has neither the range nor all steps)."""
        if dtype not in _OUT:
            raise TypeError(f"values come in bf16, fp16 or fp32, not {dtype}")
        like = self.__dict__.get("_both")
        out = (self.codes if like is None else like).new_empty(self.rows, self.k, dtype=dtype)
        if self.rows:
            status = _run(_lib.lib().plm_fp8_values, self._index, self.codes_at, self.scales_at, self.rows, self.k, self._gate_up,
                          _OUT[dtype], out.data_ptr())
            if status:
                _lib.check(status, f"plm_fp8_values({self.rows} rows of {self.k})")
        return out


class Rows(_Eight):
    """Activations ``[rows, k]`` in 8 bits, as ``quantize`` and ``rms_norm`` return them."""


class Weight(_Eight):
    """A weight ``[n, k]`` in 8 bits. ``Weight.quantize`` rounds one of 16 bits, ``Weight.from_blocks`` lays out codes and
    scales that are there already; ``Weight(codes, scales, n, k, gate_up=...)`` takes ``.codes`` and ``.scales`` of
    another (a checkpoint of this layout). ``gate_up``: a fused gate/up weight, gate rows first, for ``gate_up_silu``."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, n: int, k: int, *, gate_up: bool = False):
        _halves(n, gate_up)
        super().__init__(codes, scales, n, k)
        self.__dict__["_gate_up"] = bool(gate_up)

    @property
    def n(self) -> int:
        return self.rows

    @property
    def gate_up(self) -> bool:
        return self._gate_up

    @classmethod
    def quantize(cls, w: torch.Tensor, *, gate_up: bool = False) -> "Weight":
        """``w`` (bf16 or fp16 ``[n, k]``) rounded to 8 bits."""
        w, at, stride, code, _, n, k = _matrix(w, "w")
        if n > 1 and stride < k:
            raise ValueError("w's rows overlap")
        return cls._filled(code, n, k, at, max(stride, k), 0, gate_up, w)

    @classmethod
    def from_blocks(cls, codes: torch.Tensor, scales: torch.Tensor, *, gate_up: bool = False) -> "Weight":
        """``codes`` float8_e4m3fn ``[n, k]`` with float32 ``scales [ceil(n / 128), ceil(k / 128)]`` (of a gate/up weight the
        gate half's blocks of rows, then the up half's), powers of two in [2^-64, 2^119]: a weight is
        ``codes * scales``, finite. Reads the scales on the host; other scales are refused (round such a weight's values)."""
        if codes.dim() != 2 or codes.dtype is not E4M3 or not codes.is_cuda:
            raise ValueError(f"codes must be float8_e4m3fn [n, k] on a GPU, got {codes.dtype} {list(codes.shape)} on {codes.device}")
        n, k = codes.shape
        if n < 1 or k < 8 or k % 8:
            raise ValueError(f"codes must have rows of a multiple of 8, got {list(codes.shape)}")
        halves = _halves(n, gate_up)
        shape = (halves * -(-(n // halves) // BLOCK), -(-k // BLOCK))
        if scales.shape != shape or scales.dtype is not torch.float32 or scales.device != codes.device:
            raise ValueError(f"scales must be float32 {list(shape)} on {codes.device}, got {scales.dtype} {list(scales.shape)} on "
                             f"{scales.device}")
        _derivative(codes, "codes")
        _derivative(scales, "scales")
        if not codes.data_ptr():
            _no_memory("codes")
        if not scales.data_ptr():
            _no_memory("scales")
        scales = scales.contiguous()
        bits = scales.view(torch.int32)
        if not bool(((bits & 0x7fffff) == 0).logical_and(bits >= 63 << 23).logical_and(bits <= 246 << 23).all()):
            raise ValueError("scales must be powers of two in [2^-64, 2^119]")
        if not codes.is_contiguous() or codes.data_ptr() % 8:
            codes = codes.clone(memory_format=torch.contiguous_format)
        return cls._filled(0, n, k, codes.data_ptr(), k, scales.data_ptr(), gate_up, codes)

    @classmethod
    def _filled(cls, dtype: int, n: int, k: int, at: int, stride: int, blocks: int, gate_up: bool, like: torch.Tensor) -> "Weight":
        _halves(n, gate_up)
        if not _lib.lib().plm_fp8_codes_bytes(n, k):
            raise ValueError(f"a weight has 1 to 2^24 - 1 rows and at most 2^25 fragments, got [{n}, {k}]")
        self = cls._new(n, k, like)
        self.__dict__["_gate_up"] = bool(gate_up)
        status = _run(_lib.lib().plm_fp8_weight, self._index,
                      _lib.pack_fp8_weight(dtype, n, k, at, stride, blocks, bool(gate_up), self.codes_at, self.scales_at))
        if status:
            _lib.check(status, f"plm_fp8_weight([{n}, {k}], gate_up={gate_up})")
        return self


def _again(cls, codes: torch.Tensor, scales: torch.Tensor, rows: int, k: int, gate_up: bool):
    if not rows:
        return cls._new(rows, k, codes)
    codes = codes.view(E4M3)
    return cls(codes, scales, rows, k, gate_up=True) if gate_up else cls(codes, scales, rows, k)


def _halves(n: int, gate_up: bool) -> int:
    if gate_up and n % 32:
        raise ValueError(f"a fused gate/up weight needs a multiple of 32 rows, got {n}")
    return 2 if gate_up else 1


def quantize(x: torch.Tensor) -> Rows:
    """``x`` (bf16 or fp16 ``[rows, k]``, k a multiple of 8) in 8 bits."""
    x, at, stride, code, index, rows, k = _matrix(x, "x")
    out = Rows._new(rows, k, x)
    if rows:
        status = _run(_lib.lib().plm_fp8_rows, index,
                      _lib.pack_fp8_rows(code, rows, k, at, stride, 0, 0, 0, 0, 0, 0.0, 0, out.codes_at, out.scales_at))
        if status:
            _lib.check(status, f"plm_fp8_rows({rows} rows of {k})")
    return out


def rms_norm(x: torch.Tensor, weight: torch.Tensor | None, eps: float = 1e-6, *, residual: torch.Tensor | None = None,
             dtype: torch.dtype | None = None):
    """``t * weight / sqrt(mean(t^2) + eps)`` of ``t = x + residual``, rounded to x's type (without a residual ``t`` is
    ``x``), ``[rows, k]``: in x's type, or with ``dtype=torch.float8_e4m3fn`` as ``Rows``. With a residual the result is
    ``(norm, t)``, t being the residual of the next call. ``weight [k]`` is of x's type (None: ones); eps is in [2^-100,
    2^100]. Codes are what the exact value rounds to."""
    x, at, stride, code, index, rows, k = _matrix(x, "x")
    eight = dtype is E4M3
    if not eight and dtype is not None and dtype is not x.dtype:
        raise TypeError(f"a norm comes in its input's type or float8_e4m3fn, not {dtype}")
    if not _EPS[0] <= eps <= _EPS[1]:
        raise ValueError(f"eps must be in [2^-100, 2^100], got {eps}")
    weight_at = 0
    if weight is not None:
        if weight.dtype is not x.dtype or weight.shape != (k,) or weight.get_device() != index:
            raise ValueError(f"weight must be {x.dtype} [{k}] on cuda:{index}, got {weight.dtype} {list(weight.shape)} on {weight.device}")
        if weight.requires_grad or forward_ad._current_level >= 0:
            _derivative(weight, "weight")
        weight_at = weight.data_ptr()
        if not weight_at:
            _no_memory("weight")
        if weight_at % 16 or not weight.is_contiguous():
            weight = weight.clone(memory_format=torch.contiguous_format)
            weight_at = weight.data_ptr()
    total, total_at, residual_at, residual_stride = None, 0, 0, 0
    if residual is not None:
        if residual.shape != (rows, k) or residual.dtype is not x.dtype:
            raise ValueError(f"residual must be {x.dtype} {[rows, k]} as x is, got {residual.dtype} {list(residual.shape)}")
        residual, residual_at, residual_stride, *_ = _matrix(residual, "residual", index)
        total = x.new_empty(rows, k)
        total_at = total.data_ptr()
    if eight:
        out = Rows._new(rows, k, x)
        y_at, codes_at, scales_at = 0, out.codes_at, out.scales_at
    else:
        out = x.new_empty(rows, k)
        y_at, codes_at, scales_at = out.data_ptr(), 0, 0
    if rows:
        status = _run(_lib.lib().plm_fp8_rows, index,
                      _lib.pack_fp8_rows(code, rows, k, at, stride, 1, residual_at, residual_stride, total_at, weight_at, eps, y_at,
                                         codes_at, scales_at))
        if status:
            _lib.check(status, f"plm_fp8_rows(norm of {rows} rows of {k})")
    return out if residual is None else (out, total)


def _overlap(a: int, a_row: int, a_width: int, b: int, b_row: int, b_width: int, rows: int) -> bool:
    """Whether two matrices of as many rows share memory, by their addresses, row strides and widths in bytes; columns of one wide
    matrix do not."""
    if a + (rows - 1) * a_row + a_width <= b or b + (rows - 1) * b_row + b_width <= a:
        return False
    apart = (b - a) % a_row if a_row else 0
    return a_row != b_row or apart < a_width or apart + b_width > a_row


def _meets(begin: int, end: int, eight: _Eight) -> bool:
    """Whether [begin, end) shares memory with 8-bit rows."""
    frags, blocks = (eight.rows + 15) // 16, (eight.k + 127) // 128
    return (begin < eight.codes_at + frags * blocks * 2048 and eight.codes_at < end
            or begin < eight.scales_at + frags * ((blocks + 3) // 4) * 64 and eight.scales_at < end)


def _product(x: torch.Tensor | Rows, w: Weight, out: torch.Tensor | None, out_dtype: torch.dtype | None, act: bool) -> torch.Tensor:
    index, n, k = w._index, w.rows, w.k
    if isinstance(x, Rows):
        kind, rows, x_at, x_scales, stride, like = _lib.PLM_FP8_CODES, x.rows, x.codes_at, x.scales_at, 0, w.__dict__.get("_both")
        if out_dtype is None and out is None:
            raise ValueError("rows in 8 bits have no type of their own: out_dtype or out is needed")
        if x.k != k:
            raise ValueError(f"x must be [rows, {k}], got {[rows, x.k]}")
        if x._index != index:
            raise RuntimeError(f"x must be on the weight's GPU cuda:{index}, got cuda:{x._index}")
        if like is None:
            like = w.codes
    else:
        x, x_at, stride, code, _, rows, own = _matrix(x, "x", index)   # rounded in the call, as quantize does
        if own != k:
            raise ValueError(f"x must be [rows, {k}], got {[rows, own]}")
        like, x_scales, kind = x, 0, _IN[code]
        if out_dtype is None and out is None:
            out_dtype = x.dtype
    if out_dtype is None:
        out_dtype = out.dtype
    kind_out = _OUT.get(out_dtype)
    if kind_out is None:
        raise TypeError(f"a product comes in bf16, fp16 or fp32, not {out_dtype}")
    if rows > MOST or n > MOST:
        raise ValueError(f"a product takes up to {MOST} rows of x and of the weight, got {rows} and {n}")
    columns = n // 2 if act else n
    if out is None:
        out = like.new_empty(rows, columns, dtype=out_dtype)
        out_row = columns
    else:
        if out.shape != (rows, columns) or out.dtype is not out_dtype or out.get_device() != index or \
                (rows and (out.stride(1) != 1 and columns > 1 or out.stride(0) < columns and rows > 1)):
            raise ValueError(f"out must be a row-major {[rows, columns]} {out_dtype} tensor on cuda:{index}")
        if out.requires_grad or forward_ad._current_level >= 0:
            _derivative(out, "out")
        out_row = max(out.stride(0), columns)
        if rows:
            begin = out.data_ptr()
            end = begin + out.element_size() * ((rows - 1) * out_row + columns)
            if _meets(begin, end, w) or x_scales and _meets(begin, end, x):
                raise ValueError("out overlaps an operand, which workgroups read while others write")
        if not x_scales and rows and _overlap(x_at, 2 * stride, 2 * k, out.data_ptr(), out.element_size() * out_row,
                                              out.element_size() * columns, rows):
            raise ValueError("out overlaps x, which workgroups read while others write")
    if not rows:
        return out
    call = _lib.pack_fp8_linear(rows, n, k, kind, x_at, x_scales, stride, w.codes_at, w.scales_at, out.data_ptr(), out_row, kind_out, act)
    lib = _lib.lib()
    space, size = 0, lib.plm_fp8_linear_workspace_bytes(call)
    if size:
        work = like.new_empty(size, dtype=torch.uint8)   # rounded rows, partial sums: this call's alone
        space = work.data_ptr()
    status = _run(lib.plm_fp8_linear, index, call, space, size)
    if status:
        _lib.check(status, f"plm_fp8_linear(M={rows}, N={n}, K={k}, act={act})")
    return out


def linear(x: torch.Tensor | Rows, w: Weight, *, out: torch.Tensor | None = None,
           out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``x @ w^T`` ``[rows, n]``, summed in fp32 and rounded once to ``out_dtype``: bf16, fp16 or fp32, x's type unless given
    (``Rows`` have none). ``x`` is ``[rows, k]``, in 16 bits, which are rounded to 8 here, or ``Rows``. For 16-bit results the
    matrix instruction cuts, toward zero, each product of an eight along k at 2^-13 of two to the largest sum of two factors'
    exponents, which is 1.5e-5 to 4e-5 of a result's size (rms); for float32 every product is added whole, at up to twice the time."""
    if not isinstance(w, Weight):
        raise TypeError(f"w must be an fp8.Weight, got {type(w).__name__}")
    if w._gate_up:
        raise ValueError("a gate/up weight goes to gate_up_silu")
    return _product(x, w, out, out_dtype, False)


def gate_up_silu(x: torch.Tensor | Rows, w: Weight, *, out: torch.Tensor | None = None,
                 out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``silu(g) * u`` of the halves of ``x @ w^T``, ``[rows, n / 2]``: in fp32 up to the one rounding to ``out_dtype``
    (``fast_gemm.gate_up_silu`` rounds the projections and the activation on the way), the sums as ``linear``'s, the
    activation good to 2^-20 of its value for gates down to -174. ``w`` is a gate/up weight."""
    if not isinstance(w, Weight):
        raise TypeError(f"w must be an fp8.Weight, got {type(w).__name__}")
    if not w._gate_up:
        raise ValueError("gate_up_silu needs a weight made with gate_up=True")
    return _product(x, w, out, out_dtype, True)


def llama_mlp(x: torch.Tensor | Rows, gate_up: Weight, down: Weight, *, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """A gated MLP over 8-bit weights, ``down(silu(g) * u)``: the 8-bit form of ``fast_gemm.llama_mlp``. The activation is
    rounded to ``out_dtype`` (bf16 or fp16, x's type unless given) and from there to 8 bits."""
    act = gate_up_silu(x, gate_up, out_dtype=out_dtype)
    return linear(act, down)
