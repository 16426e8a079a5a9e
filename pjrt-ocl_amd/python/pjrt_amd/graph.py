"""Tensor-graph builder: emits VMProgram tensor instructions.

This is the instruction-selection layer of the lowering: every StableHLO op the
front-end understands becomes one or more calls here, and hand-written programs
(tests, benchmarks) use it directly.  The instructions it emits follow the
reference lowering's encodings op for op (python/pjrt_ocl/ops/*.py handlers,
lowering.py:286-331), so the resulting bytes are a reference-format program.

    g = Graph()
    x = g.input((8, 4), "f32")
    y = g.add(x, g.const(np.ones((8, 4), np.float32)))
    g.output(y)
    prog = g.build()              # VMProgram (tensor sections, arena laid out)
"""
from __future__ import annotations

import dataclasses
import fractions
import math

import numpy as np

from . import vmprogram as V


def _prod(shape) -> int:
    return int(math.prod(shape)) if len(shape) else 1


def _row_major_strides(shape):
    st, acc = [0] * len(shape), 1
    for d in range(len(shape) - 1, -1, -1):
        st[d] = acc
        acc *= shape[d]
    return st


def _dt(d) -> int:
    if isinstance(d, str):
        return V.DT_BY_NAME[d]
    return int(d)


@dataclasses.dataclass(frozen=True)
class Tensor:
    buf: int
    shape: tuple
    dtype: int
    # optional strided view over ``buf`` (aux word offset + 1); set only on
    # values produced by ``view`` and consumed by ops that accept views
    view: int = 0

    @property
    def n(self) -> int:
        return _prod(self.shape)


class GraphError(ValueError):
    pass


@dataclasses.dataclass(frozen=True)
class PagedCache:
    """Keys and values of many sequences in pages that the caller owns and the
    program writes in place (``Graph.paged_cache``): pages [N, heads, page, head_dim]
    of one dtype, or i8 with one f32 scale per (page, head, position)."""
    k: Tensor
    v: Tensor
    k_scale: Tensor | None
    v_scale: Tensor | None

    @property
    def dims(self) -> tuple:
        return self.k.shape


@dataclasses.dataclass(frozen=True)
class PagedBatch:
    """The rows of a step (``Graph.paged_batch``): sequence s's new tokens are rows
    cu[s] .. cu[s + 1] - 1, its length with them is lens[s], and position p of it
    lies in page table[s, p // page].  cu does not fall; a sequence that has rows
    outside the step's is served as one whose length does not fit its rows."""
    cu: Tensor
    lens: Tensor
    table: Tensor


def rotary_frequencies(rot: int, theta: float = 10000.0, factor: float = 1.0, original: int = 0,
                       low: float = 1.0, high: float = 32.0) -> np.ndarray:
    """Radians per position of each of the rot / 2 channel pairs, f64:
    theta^(-2 i / rot).  ``factor`` > 1 stretches positions for contexts longer than
    the ``original`` one the model was trained on: frequencies that turn fewer than
    ``low`` times over it are divided by the factor, those of more than ``high`` turns
    are kept, and the ones between are blended linearly in their turns;
    with ``original`` 0 every frequency is divided."""
    if rot < 2 or rot % 2:
        raise GraphError("rotary_frequencies: rot is even and at least 2")
    if not (theta > 0 and factor >= 1.0 and original >= 0 and 0 <= low < high):
        raise GraphError("rotary_frequencies: theta > 0, factor >= 1, original >= 0 and 0 <= low < high")
    f = float(theta) ** (-2.0 * np.arange(rot // 2, dtype=np.float64) / rot)
    if factor == 1.0:
        return f
    if not original:
        return f / factor
    keep = np.clip((original * f / (2.0 * np.pi) - low) / (high - low), 0.0, 1.0)
    return f * keep + f / factor * (1.0 - keep)


def _two_pi_inverse_2_192() -> int:
    """floor(2^192 / (2 pi)) by Machin's formula pi = 16 atan(1/5) - 4 atan(1/239)."""
    one = 1 << 256

    def atan_inv(k):
        total, power, n = 0, one // k, 1
        while power:
            total += power // n if n % 4 == 1 else -(power // n)
            power //= k * k
            n += 2
        return total
    pi = 16 * atan_inv(5) - 4 * atan_inv(239)          # pi 2^256
    return (1 << 447) // pi                            # 2^192 / (2 pi)


_INV_2PI = fractions.Fraction(_two_pi_inverse_2_192(), 1 << 192)


def turn_words(inv_freq) -> np.ndarray:
    """[R, 2] u32: each frequency (radians per position) as the low and high words of
    its 64-bit fixed-point fraction of a turn, so that position * frequency modulo one
    turn is one integer product, exact to 2^-33 turns for every 32-bit position."""
    out = np.empty((len(inv_freq), 2), np.uint32)
    for i, f in enumerate(inv_freq):
        w = round(fractions.Fraction(float(f)) * _INV_2PI * (1 << 64)) & ((1 << 64) - 1)
        out[i] = (w & 0xFFFFFFFF, w >> 32)
    return out


class Graph:
    def __init__(self):
        self.buffers: list = []         # [(n_elems, dtype)]
        self.instrs: list = []          # root instruction list being built
        self.regions: list = []         # finished sub-lists appended at build
        self.aux: list = []
        self.consts: list = []          # [(buf, bytes)]
        self.inputs: list = []
        self.outputs: list = []
        self._stack: list = []          # instruction lists under construction
        self._disjoint = 0
        self.aliases: dict = {}         # buffer -> (parent buffer, byte offset)
        self.states: set = set()        # inputs written in place

    # ---- buffers / io -----------------------------------------------------
    def _new(self, shape, dtype) -> Tensor:
        shape = tuple(int(s) for s in shape)
        self.buffers.append((_prod(shape), _dt(dtype)))
        return Tensor(len(self.buffers) - 1, shape, _dt(dtype))

    def input(self, shape, dtype="f32") -> Tensor:
        t = self._new(shape, dtype)
        self.inputs.append(t)
        return t

    def state(self, shape, dtype="f32") -> Tensor:
        """An input that the program's tasks write in place: memory the caller owns
        and keeps between runs, such as a cache.  It takes no arena bytes, so it may
        be of any size, and must not overlap another input or output of the run."""
        t = self.input(shape, dtype)
        self.states.add(t.buf)
        return t

    def const(self, value, dtype=None) -> Tensor:
        arr = np.asarray(value)
        if dtype is None:
            dtype = {np.float32: V.DT_F32, np.int32: V.DT_I32,
                     np.uint32: V.DT_U32, np.bool_: V.DT_BOOL,
                     np.int64: V.DT_I64, np.float64: V.DT_F64,
                     np.float16: V.DT_F16}.get(arr.dtype.type, V.DT_F32)
        dt = _dt(dtype)
        if dt == V.DT_BF16 and arr.dtype != np.uint16:
            raw = V.f32_to_bf16(arr.astype(np.float32))
        elif dt == V.DT_BOOL:
            raw = arr.astype(np.uint8)
        else:
            raw = arr.astype(V.DT_NUMPY[dt])
        t = self._new(arr.shape, dt)
        self.consts.append((t.buf, np.ascontiguousarray(raw).tobytes()))
        return t

    def scalar(self, v, dtype="f32") -> Tensor:
        dt = _dt(dtype)
        if dt == V.DT_BF16:
            return self.const(np.asarray(v, np.float32), dt)
        return self.const(np.asarray(v, V.DT_NUMPY[dt] if dt != V.DT_BOOL else np.uint8), dt)

    def output(self, *ts: Tensor) -> None:
        for t in ts:
            if t.buf in self.states:
                raise GraphError("a state buffer is updated in place and is no output")
            self.outputs.append(t)

    def add_aux(self, words) -> int:
        off = len(self.aux)
        self.aux.extend(int(w) & 0xFFFFFFFF for w in words)
        return off

    def emit(self, ins: V.Instr) -> None:
        (self._stack[-1] if self._stack else self.instrs).append(ins)

    # ---- views (strided reads folded into consumers) ------------------------
    def view(self, src: Tensor, out_shape, in_strides, src_off=0) -> Tensor:
        """A strided view ``out[i] = src[src_off + sum_d coord_d(i) * stride_d]``
        that elementwise and matmul consumers read in place."""
        rank = len(out_shape)
        off = self.add_aux([rank] + list(out_shape) + list(in_strides) + [src_off])
        return Tensor(src.buf, tuple(out_shape), src.dtype, view=off + 1)

    def broadcast_view(self, src: Tensor, out_shape, dims) -> Tensor:
        """broadcast_in_dim as a view: src axis k maps to out axis dims[k]."""
        st = _row_major_strides(src.shape)
        in_strides = [0] * len(out_shape)
        for k, d in enumerate(dims):
            if src.shape[k] != 1:
                in_strides[d] = st[k]
        return self.view(src, out_shape, in_strides)

    def transpose_view(self, src: Tensor, perm) -> Tensor:
        st = _row_major_strides(src.shape)
        return self.view(src, [src.shape[p] for p in perm], [st[p] for p in perm])

    def alias(self, src: Tensor, elem_off: int, shape) -> Tensor:
        """A contiguous slice of ``src`` as a buffer of its own that shares src's
        memory (no copy): elements [elem_off, elem_off + prod(shape)).  The
        scheduler orders accesses to overlapping buffers like accesses to one."""
        src = self.materialize(src)
        shape = tuple(int(x) for x in shape)
        if elem_off < 0 or elem_off + _prod(shape) > src.n:
            raise GraphError("alias outside its source")
        byte_off = elem_off * V.DT_SIZE[src.dtype]
        if byte_off % 16:
            raise GraphError("alias offset must keep 16-byte alignment")
        if src.buf in self.states:
            raise GraphError("alias of a state buffer")
        parent, base = self.aliases.get(src.buf, (src.buf, 0))
        t = self._new(shape, src.dtype)
        self.aliases[t.buf] = (parent, base + byte_off)
        return t

    def materialize(self, t: Tensor) -> Tensor:
        if not t.view:
            return t
        dst = self._new(t.shape, t.dtype)
        self.emit(V.Instr(V.OP_GATHER_STRIDED, dst=dst.buf, a=t.buf, n=t.n,
                          aux=t.view - 1))
        return dst

    # ---- shape ops ------------------------------------------------------------
    def reshape(self, t: Tensor, shape) -> Tensor:
        t = self.materialize(t)
        if _prod(shape) != t.n:
            raise GraphError("reshape changes element count")
        return Tensor(t.buf, tuple(shape), t.dtype)

    def gather(self, src: Tensor, out_shape, in_strides, src_off=0) -> Tensor:
        return self.materialize(self.view(self.materialize(src), out_shape,
                                          in_strides, src_off))

    def broadcast(self, src: Tensor, out_shape, dims) -> Tensor:
        return self.materialize(self.broadcast_view(self.materialize(src),
                                                    out_shape, dims))

    def transpose(self, src: Tensor, perm) -> Tensor:
        return self.materialize(self.transpose_view(self.materialize(src), perm))

    def slice(self, src: Tensor, starts, limits, strides=None) -> Tensor:
        src = self.materialize(src)
        strides = strides or [1] * len(starts)
        st = _row_major_strides(src.shape)
        out_shape = [max(0, -(-(l - s) // k)) for s, l, k in zip(starts, limits, strides)]
        return self.gather(src, out_shape, [st[d] * strides[d] for d in range(len(st))],
                           sum(starts[d] * st[d] for d in range(len(st))))

    def scatter_into(self, dst: Tensor, src: Tensor, out_strides, out_off,
                     disjoint: int = 0) -> None:
        src = self.materialize(src)
        rank = len(src.shape)
        off = self.add_aux([rank] + list(src.shape) + list(out_strides) + [out_off])
        self.emit(V.Instr(V.OP_SCATTER, dst=dst.buf, a=src.buf, n=src.n, aux=off,
                          disjoint=disjoint))

    def concatenate(self, parts, axis: int) -> Tensor:
        shape = list(parts[0].shape)
        shape[axis] = sum(p.shape[axis] for p in parts)
        out = self._new(shape, parts[0].dtype)
        ost = _row_major_strides(shape)
        self._disjoint += 1
        pos = 0
        for p in parts:
            self.scatter_into(out, p, ost, pos * ost[axis], self._disjoint)
            pos += p.shape[axis]
        return out

    # ---- elementwise ------------------------------------------------------------
    def _binop(self, op, a: Tensor, b: Tensor, out_dtype=None) -> Tensor:
        if a.shape != b.shape:
            raise GraphError(f"shape mismatch {a.shape} vs {b.shape}")
        dt = a.dtype if out_dtype is None else _dt(out_dtype)
        viewable = a.dtype == V.DT_F32 and op in (
            V.OP_ADD_F32, V.OP_MUL_F32, V.OP_SUB_F32, V.OP_DIV_F32,
            V.OP_MAX_F32, V.OP_MIN_F32, V.OP_POW_F32)
        if not viewable:
            a, b = self.materialize(a), self.materialize(b)
        dst = self._new(a.shape, dt)
        self.emit(V.Instr(op, dst=dst.buf, a=a.buf, b=b.buf, n=a.n, imm=a.view,
                          imm2=b.view))
        return dst

    def _unop(self, op, a: Tensor, out_dtype=None) -> Tensor:
        viewable = a.dtype == V.DT_F32 and op in (
            V.OP_COPY_F32, V.OP_NEG_F32, V.OP_EXP_F32, V.OP_LOG_F32,
            V.OP_SQRT_F32, V.OP_RSQRT_F32, V.OP_TANH_F32, V.OP_ABS_F32,
            V.OP_GELU)
        if not viewable:
            a = self.materialize(a)
        dst = self._new(a.shape, a.dtype if out_dtype is None else out_dtype)
        self.emit(V.Instr(op, dst=dst.buf, a=a.buf, n=a.n, imm=a.view))
        return dst

    def add(self, a, b): return self._binop(V.OP_ADD_F32, a, b)
    def mul(self, a, b): return self._binop(V.OP_MUL_F32, a, b)
    def sub(self, a, b): return self._binop(V.OP_SUB_F32, a, b)
    def div(self, a, b): return self._binop(V.OP_DIV_F32, a, b)
    def maximum(self, a, b): return self._binop(V.OP_MAX_F32, a, b)
    def minimum(self, a, b): return self._binop(V.OP_MIN_F32, a, b)
    def pow(self, a, b): return self._binop(V.OP_POW_F32, a, b)
    def atan2(self, a, b): return self._binop(V.OP_ATAN2_F32, a, b)
    def remainder(self, a, b): return self._binop(V.OP_REMAINDER_F32, a, b)
    def bit_and(self, a, b): return self._binop(V.OP_AND, a, b)
    def bit_or(self, a, b): return self._binop(V.OP_OR, a, b)
    def bit_xor(self, a, b): return self._binop(V.OP_XOR, a, b)
    def shl(self, a, b): return self._binop(V.OP_SHL, a, b)
    def shr_l(self, a, b): return self._binop(V.OP_SHR_L, a, b)
    def shr_a(self, a, b): return self._binop(V.OP_SHR_A, a, b)

    def unary(self, name: str, a: Tensor) -> Tensor:
        op = {"copy": V.OP_COPY_F32, "neg": V.OP_NEG_F32, "exp": V.OP_EXP_F32,
              "log": V.OP_LOG_F32, "sqrt": V.OP_SQRT_F32,
              "rsqrt": V.OP_RSQRT_F32, "tanh": V.OP_TANH_F32,
              "abs": V.OP_ABS_F32, "floor": V.OP_FLOOR_F32,
              "ceil": V.OP_CEIL_F32, "sign": V.OP_SIGN_F32,
              "log1p": V.OP_LOG1P_F32, "expm1": V.OP_EXPM1_F32,
              "cbrt": V.OP_CBRT_F32, "sin": V.OP_SIN_F32, "cos": V.OP_COS_F32,
              "tan": V.OP_TAN_F32, "rint": V.OP_ROUND_NEAREST_EVEN_F32,
              "round": V.OP_ROUND_NEAREST_AFZ_F32, "not": V.OP_NOT,
              "gelu": V.OP_GELU}[name]
        return self._unop(op, a)

    def gelu(self, a): return self._unop(V.OP_GELU, a)

    def affine(self, a: Tensor, s: float, t: float) -> Tensor:
        a = self.materialize(a)
        dst = self._new(a.shape, a.dtype)
        self.emit(V.Instr(V.OP_AFFINE_F32, dst=dst.buf, a=a.buf, n=a.n,
                          imm=V.f32_bits(s), imm2=V.f32_bits(t)))
        return dst

    def fill(self, shape, value, dtype="f32") -> Tensor:
        dt = _dt(dtype)
        dst = self._new(shape, dt)
        if dt in (V.DT_F32, V.DT_F16, V.DT_BF16, V.DT_F64):
            bits = V.f32_bits(value)
        else:
            bits = int(value) & 0xFFFFFFFF
        self.emit(V.Instr(V.OP_FILL_F32, dst=dst.buf, n=dst.n, imm=bits))
        return dst

    def iota_flat(self, n: int, dtype="f32") -> Tensor:
        dst = self._new((n,), dtype)
        self.emit(V.Instr(V.OP_IOTA_F32, dst=dst.buf, n=n))
        return dst

    def iota(self, shape, dim: int, dtype="i32") -> Tensor:
        dst = self._new(shape, dtype)
        off = self.add_aux([len(shape)] + list(shape) + [dim])
        self.emit(V.Instr(V.OP_IOTA_DIM, dst=dst.buf, n=dst.n, aux=off))
        return dst

    def compare(self, a: Tensor, b: Tensor, pred: str) -> Tensor:
        a, b = self.materialize(a), self.materialize(b)
        p = {"EQ": 0, "NE": 1, "LT": 2, "LE": 3, "GT": 4, "GE": 5}[pred]
        dst = self._new(a.shape, V.DT_BOOL)
        self.emit(V.Instr(V.OP_CMP_F32, dst=dst.buf, a=a.buf, b=b.buf, n=a.n, imm=p))
        return dst

    def select(self, pred: Tensor, on_true: Tensor, on_false: Tensor) -> Tensor:
        pred, on_true, on_false = map(self.materialize, (pred, on_true, on_false))
        dst = self._new(on_true.shape, on_true.dtype)
        self.emit(V.Instr(V.OP_SELECT_F32, dst=dst.buf, a=on_true.buf,
                          b=on_false.buf, n=dst.n, imm=pred.buf))
        return dst

    def convert(self, a: Tensor, dtype) -> Tensor:
        a = self.materialize(a)
        dst = self._new(a.shape, dtype)
        self.emit(V.Instr(V.OP_CONVERT, dst=dst.buf, a=a.buf, n=a.n))
        return dst

    def bitcast(self, a: Tensor, dtype) -> Tensor:
        a = self.materialize(a)
        if V.DT_SIZE[a.dtype] != V.DT_SIZE[_dt(dtype)]:
            raise GraphError("bitcast between different widths")
        dst = self._new(a.shape, dtype)
        self.emit(V.Instr(V.OP_BITCAST, dst=dst.buf, a=a.buf, n=a.n))
        return dst

    def is_finite(self, a: Tensor) -> Tensor:
        a = self.materialize(a)
        dst = self._new(a.shape, V.DT_BOOL)
        self.emit(V.Instr(V.OP_IS_FINITE, dst=dst.buf, a=a.buf, n=a.n))
        return dst

    def lts(self, a: Tensor, b: Tensor) -> Tensor:
        dst = self._new((), V.DT_F32)
        self.emit(V.Instr(V.OP_LTS_F32, dst=dst.buf, a=a.buf, b=b.buf, n=1))
        return dst

    # ---- reductions ------------------------------------------------------------
    def reduce_all(self, a: Tensor, kind: int, ew_ts: int = 4096) -> Tensor:
        from .scheduler import red_chunk
        a = self.materialize(a)
        chunk = red_chunk(a.n, ew_ts)
        nparts = max(1, math.ceil(a.n / chunk))
        part = self._new((nparts,), a.dtype)
        self.emit(V.Instr(V.OP_REDUCE, dst=part.buf, a=a.buf, n=a.n, imm=kind))
        out = self._new((), a.dtype)
        self.emit(V.Instr(V.OP_REDUCE, dst=out.buf, a=part.buf, n=nparts,
                          imm=(1 << 3) | kind))
        return out

    def reduce_last(self, a: Tensor, kind: int) -> Tensor:
        a = self.materialize(a)
        seg = a.shape[-1]
        dst = self._new(a.shape[:-1], a.dtype)
        self.emit(V.Instr(V.OP_REDUCE_SEG, dst=dst.buf, a=a.buf, n=dst.n,
                          imm=(kind << 28) | seg))
        return dst

    def reduce_axis(self, a: Tensor, axis: int, kind: int) -> Tensor:
        a = self.materialize(a)
        if axis == len(a.shape) - 1:
            return self.reduce_last(a, kind)
        outer = _prod(a.shape[:axis])
        red = a.shape[axis]
        inner = _prod(a.shape[axis + 1:])
        dst = self._new(a.shape[:axis] + a.shape[axis + 1:], a.dtype)
        self.emit(V.Instr(V.OP_REDUCE_STRIDED, dst=dst.buf, a=a.buf,
                          n=outer * inner, imm=(kind << 28) | red, imm2=inner))
        return dst

    def argmax_last(self, a: Tensor, index_dtype="i32"):
        """(max value, first index of the max) over the last axis."""
        a = self.materialize(a)
        seg = a.shape[-1]
        idx = self._new(a.shape[:-1], index_dtype)
        val = self._new(a.shape[:-1], a.dtype)
        self.emit(V.Instr(V.OP_ARGMAX_SEG, dst=idx.buf, a=a.buf, b=val.buf,
                          n=idx.n, imm=seg))
        return val, idx

    def softmax_last(self, a: Tensor, out_dtype=None) -> Tensor:
        a = self.materialize(a)
        dst = self._new(a.shape, a.dtype if out_dtype is None else out_dtype)
        self.emit(V.Instr(V.OP_SOFTMAX, dst=dst.buf, a=a.buf,
                          n=a.n // a.shape[-1], imm=a.shape[-1]))
        return dst

    def layernorm_core(self, a: Tensor, eps: float) -> Tensor:
        a = self.materialize(a)
        dst = self._new(a.shape, a.dtype)
        self.emit(V.Instr(V.OP_LAYERNORM, dst=dst.buf, a=a.buf,
                          n=a.n // a.shape[-1], imm=a.shape[-1],
                          imm2=V.f32_bits(eps)))
        return dst

    def layernorm(self, a: Tensor, gamma: Tensor | None, beta: Tensor | None,
                  eps: float, gelu: bool = False, out_dtype=None) -> Tensor:
        """Fused row layernorm (two-pass variance) with optional per-column
        affine, tanh-GELU and output dtype conversion: one read, one write."""
        a = self.materialize(a)
        flags = V.LN_TWO_PASS | (V.LN_GELU if gelu else 0)
        if gamma is not None:
            flags |= V.LN_AFFINE
            gamma, beta = self.materialize(gamma), self.materialize(beta)
        off = self.add_aux([flags, beta.buf if gamma is not None else 0])
        dst = self._new(a.shape, a.dtype if out_dtype is None else out_dtype)
        self.emit(V.Instr(V.OP_LAYERNORM_AFFINE, dst=dst.buf, a=a.buf,
                          b=gamma.buf if gamma is not None else a.buf,
                          n=a.n // a.shape[-1], imm=a.shape[-1],
                          imm2=V.f32_bits(eps), aux=off,
                          reads_hint=(beta.buf,) if gamma is not None else ()))
        return dst

    # ---- contractions -------------------------------------------------------------
    def dot(self, a: Tensor, b: Tensor, out_dtype="f32", epilogue=None,
            residual: Tensor | None = None, tile: int = 0) -> Tensor:
        """C[G,M,N] = A[G,M,K] @ B[G,K,N]; leading dims of a 2-D-weight matmul
        fold into M.  ``a``/``b`` may be views (folded transposes).  The
        epilogue is a list of (kind, src, s, t) micro-ops applied before the
        store (src 0: unary, 1: residual per element, 2: residual per column,
        3: the constant s -- this build's extension, e.g. relu as (MAX, 3, 0, 0))."""
        if len(b.shape) == 2:
            G = 1
            K = a.shape[-1]
            M = _prod(a.shape[:-1])
            N = b.shape[1]
            out_shape = a.shape[:-1] + (N,)
        else:
            G = _prod(a.shape[:-2])
            M, K = a.shape[-2], a.shape[-1]
            N = b.shape[-1]
            if _prod(b.shape[:-2]) != G:
                raise GraphError("batch mismatch")
            out_shape = a.shape[:-1] + (N,)
        if b.shape[-2] != K:
            raise GraphError(f"contracting mismatch {a.shape} @ {b.shape}")
        if N > 0xFFFF or K > 0xFFFF:
            raise GraphError("N/K exceed the 16-bit packing of the DOT encoding")
        dst = self._new(out_shape, out_dtype)
        epi = 0
        if epilogue:
            words = [len(epilogue)]
            for kind, src, s, t in epilogue:
                words += [kind, src, V.f32_bits(s), V.f32_bits(t)]
            epi = self.add_aux(words) + 1
        ins = V.Instr(V.OP_DOT, dst=dst.buf, a=a.buf, b=b.buf, n=M,
                      imm=(N << 16) | K, imm2=G, aview=a.view, bview=b.view,
                      epi=epi, epi_res=residual.buf if residual is not None else 0,
                      mma_tile=tile)
        if a.view or b.view or epi:
            # mirror of the in-memory view/epilogue fields in an aux header so
            # re-parsed bytes keep them (lowering.py:2455-2466)
            ins.aux = self.add_aux([a.view, b.view, epi,
                                    residual.buf if residual is not None else 0])
        if residual is not None:
            ins.reads_hint = (residual.buf,)
        self.emit(ins)
        return dst

    def flash_attention(self, q: Tensor, k: Tensor, v: Tensor, scale: float,
                        causal: bool, out_dtype=None) -> Tensor:
        """softmax(scale * Q K^T [causal]) V over heads.  q: [..., T, hd],
        k/v: [..., C, hd] (same leading dims, flattened into H).  K is read as
        the matmul B operand [H, hd, C] through a transpose view, as the
        reference's fused op does (ops/attention.py:53-64)."""
        q, k, v = self.materialize(q), self.materialize(k), self.materialize(v)
        H = _prod(q.shape[:-2])
        T, hd = q.shape[-2], q.shape[-1]
        C = k.shape[-2]
        kt = self.view(k, (H, hd, C), (C * hd, 1, hd))   # [H,hd,C] <- [H,C,hd]
        desc = self.add_aux([H, T, C, hd, V.f32_bits(scale), int(causal),
                             0, kt.view, 0])
        dst = self._new(q.shape, q.dtype if out_dtype is None else out_dtype)
        self.emit(V.Instr(V.OP_FLASH_ATTN, dst=dst.buf, a=q.buf, b=k.buf, n=H,
                          imm=T, aux=desc, imm2=v.buf))
        return dst

    def decode_attention(self, q: Tensor, k: Tensor, v: Tensor, cache_kt: Tensor,
                         cache_v: Tensor, pos: Tensor, scale: float, krow: bool = False,
                         masked: bool = False) -> Tensor:
        """One decode step of attention per head (extension opcode
        OP_DECODE_ATTN): the keys are the cache prefix K^T[h, :, :pos] and the
        step's own key k[h], the values V[h, :pos] and v[h], so the step reads
        its new key/value straight from where they were computed and the cache
        update can run beside the next matmul.  q, k, v: [H, hd] (any shape of
        H * hd elements); cache_kt: [H, hd, C], or the key rows [H, C, hd] with
        ``krow``; cache_v: [H, C, hd]; pos: i32 scalar,
        clamped to [0, C].  All float operands share one dtype; the output
        [H, hd] has it too.  Equals the decomposed dot -> (mask beyond pos) ->
        softmax -> dot chain with pos's column of the cache holding k and v.
        ``masked``: that chain as a decoder writes it after storing k and v at
        pos: pos is clamped to [0, C - 1] like the store, and a negative pos
        leaves no key, so the output is NaN."""
        if cache_kt.view or cache_v.view:
            raise GraphError("decode_attention: caches must be plain buffers")
        q, k, v = self.materialize(q), self.materialize(k), self.materialize(v)
        if len(cache_kt.shape) != 3 or len(cache_v.shape) != 3:
            raise GraphError("decode_attention: caches are [H, hd, C] and [H, C, hd]")
        if krow:
            H, C, hd = cache_kt.shape
        else:
            H, hd, C = cache_kt.shape
        if cache_v.shape != (H, C, hd):
            raise GraphError(f"decode_attention: V cache {cache_v.shape} != {(H, C, hd)}")
        for name, t in (("q", q), ("k", k), ("v", v)):
            if t.n != H * hd:
                raise GraphError(f"decode_attention: {name} has {t.n} elements, want {H * hd}")
        dts = {t.dtype for t in (q, k, v, cache_kt, cache_v)}
        if len(dts) != 1 or next(iter(dts)) not in (V.DT_F32, V.DT_F16, V.DT_BF16):
            raise GraphError("decode_attention: q, k, v and the caches share one float dtype")
        if pos.n != 1 or pos.dtype != V.DT_I32:
            raise GraphError("decode_attention: pos is an i32 scalar")
        if hd % 8 or hd > 256 or C % 8 or C > 0xFFFF:
            raise GraphError("decode_attention: hd and C must be multiples of 8 (hd <= 256)")
        dst = self._new((H, hd), q.dtype)
        desc = self.add_aux([hd | int(krow) << 16 | int(masked) << 17, k.buf, v.buf, pos.buf,
                             V.f32_bits(scale)])
        self.emit(V.Instr(V.OP_DECODE_ATTN, dst=dst.buf, a=q.buf, b=cache_kt.buf, n=H,
                          imm=C, aux=desc, imm2=cache_v.buf,
                          reads_hint=(cache_v.buf, k.buf, v.buf, pos.buf)))
        return dst

    # ---- rotary positions and the paged cache (extensions) ------------------------
    def _heads_view(self, t: Tensor, what: str) -> tuple:
        """(buffer, row stride, head stride, offset) of [rows, heads, head_dim] rows:
        a plain tensor, or a view of one whose last stride is 1."""
        if len(t.shape) != 3:
            raise GraphError(f"{what}: [rows, heads, head_dim], got {t.shape}")
        if not t.view:
            return t.buf, t.shape[1] * t.shape[2], t.shape[2], 0
        w = self.aux[t.view - 1:t.view - 1 + 8]
        w = [x - (1 << 32) if x >= 1 << 31 else x for x in w]
        (rs, hs, cs), off = w[4:7], w[7]
        if cs != 1 and t.shape[2] > 1 or min(rs, hs, off) < 0:
            raise GraphError(f"{what}: a view needs contiguous channels and strides of at least 0")
        return t.buf, rs, hs, off

    def _floats(self, what: str, *ts: Tensor) -> int:
        dts = {t.dtype for t in ts}
        if len(dts) != 1 or next(iter(dts)) not in (V.DT_F32, V.DT_F16, V.DT_BF16):
            raise GraphError(f"{what}: operands share one of f32, f16 and bf16")
        return next(iter(dts))

    def _rotary_args(self, what, x, pos, inv_freq, weight, eps):
        T, H, hd = x.shape
        inv_freq = [float(f) for f in inv_freq]
        rot = 2 * len(inv_freq)
        if hd % 2 or not 2 <= hd <= 256 or not 2 <= rot <= hd:
            raise GraphError(f"{what}: head_dim {hd} is even and at most 256, with 2 .. head_dim rotated channels, not {rot}")
        if T < 1 or H < 1:
            raise GraphError(f"{what}: no rows")
        if not all(math.isfinite(f) for f in inv_freq):
            raise GraphError(f"{what}: frequencies are finite")
        if pos.shape != (T,) or pos.dtype != V.DT_I32 or pos.view:
            raise GraphError(f"{what}: positions are i32 [{T}]")
        if weight is not None and (weight.shape != (hd,) or weight.dtype != V.DT_F32 or weight.view):
            raise GraphError(f"{what}: the norm's weight is f32 [{hd}]")
        if not (eps >= 0.0 and math.isfinite(eps)):
            raise GraphError(f"{what}: eps is finite and at least 0")
        return rot, self.const(turn_words(inv_freq), "u32")

    def rotary(self, x: Tensor, pos: Tensor, inv_freq, weight: Tensor | None = None, eps: float = 1e-6,
               interleaved: bool = False, magnitude: float = 1.0, inverse: bool = False) -> Tensor:
        """Rotary positions of the heads of x [T, H, hd], a tensor or a view of a wider
        row (queries inside a fused projection): channel pair i of row t is rotated by
        pos[t] * inv_freq[i] radians and scaled by ``magnitude``, channels past the
        2 len(inv_freq) rotated ones pass.  Pairs are (i, i + R) of R = len(inv_freq), or
        (2 i, 2 i + 1) with ``interleaved``.  With ``weight`` (f32 [hd]) each head is
        first normalised: x / sqrt(mean(x^2) + eps) * weight, in the same pass.
        ``inverse`` rotates back, which is the gradient of the rotation without a
        norm.  Angles are exact to 2^-32 turns at every 32-bit position; arithmetic is
        f32, rounded once.  Returns [T, H, hd] of x's dtype."""
        what = "rotary"
        buf, rs, hs, off = self._heads_view(x, what)
        dt = self._floats(what, x)
        rot, freq = self._rotary_args(what, x, pos, inv_freq, weight, eps)
        T, H, hd = x.shape
        flags = interleaved * V.ROT_INTERLEAVED | (weight is not None) * V.ROT_NORM | inverse * V.ROT_INVERSE
        desc = self.add_aux([T, H, hd, rot, flags, V.f32_bits(eps), V.f32_bits(magnitude), rs, hs, off, 0, 0, 0,
                             freq.buf])
        dst = self._new(x.shape, dt)
        wb = weight.buf if weight is not None else buf
        self.emit(V.Instr(V.OP_ROTARY, dst=dst.buf, a=buf, b=wb, n=T, imm=H, aux=desc, imm2=pos.buf,
                          reads_hint=(pos.buf, freq.buf)))
        return dst

    def rotary_grad(self, dy: Tensor, x: Tensor, pos: Tensor, inv_freq, weight: Tensor | None = None,
                    eps: float = 1e-6, interleaved: bool = False, magnitude: float = 1.0):
        """Gradients of ``rotary`` at x: (dx of x's dtype, dweight f32 [hd], or None
        without a norm).  Sums over rows are f32, in an order that depends on the
        shapes alone."""
        what = "rotary_grad"
        if dy.shape != x.shape:
            raise GraphError(f"{what}: dy {dy.shape} and x {x.shape}")
        dt = self._floats(what, dy, x)
        if weight is None:
            return self.rotary(dy, pos, inv_freq, interleaved=interleaved, magnitude=magnitude, inverse=True), None
        (db, drs, dhs, doff), (xb, xrs, xhs, xoff) = self._heads_view(dy, what), self._heads_view(x, what)
        rot, freq = self._rotary_args(what, x, pos, inv_freq, weight, eps)
        T, H, hd = x.shape
        flags = interleaved * V.ROT_INTERLEAVED | V.ROT_NORM
        dst = self._new(x.shape, dt)
        workers = rotary_grad_workers(T, H)
        part, dw = self._new((workers, hd), V.DT_F32), self._new((hd,), V.DT_F32)
        desc = self.add_aux([T, H, hd, rot, flags, V.f32_bits(eps), V.f32_bits(magnitude), drs, dhs, doff,
                             xrs, xhs, xoff, freq.buf, weight.buf, part.buf, workers, dw.buf])
        self.emit(V.Instr(V.OP_ROTARY_GRAD, dst=dst.buf, a=db, b=xb, n=T, imm=H, aux=desc, imm2=pos.buf,
                          reads_hint=(pos.buf, freq.buf, weight.buf)))
        return dst, dw

    def paged_cache(self, pages: int, heads: int, page: int, head_dim: int, dtype="bf16") -> PagedCache:
        """State inputs of a cache of ``pages`` pages of ``page`` positions: k and v
        pages [pages, heads, page, head_dim], and for i8 the scales [pages, heads,
        page] f32 of k and of v, in this order.  Any page size; head_dim a multiple of
        8 up to 256."""
        dt = _dt(dtype)
        if dt not in (V.DT_F32, V.DT_F16, V.DT_BF16, V.DT_I8):
            raise GraphError("paged_cache: pages are f32, f16, bf16 or i8")
        if pages < 1 or heads < 1 or page < 1 or head_dim % 8 or not 8 <= head_dim <= 256:
            raise GraphError("paged_cache: at least one page, head and position; head_dim a multiple of 8 up to 256")
        if page > 1 << 16 or pages >= 1 << 31 or heads > 1 << 16 or pages * heads * page >= 1 << 32:
            raise GraphError("paged_cache: too large")
        shape = (pages, heads, page, head_dim)
        k, v = self.state(shape, dt), self.state(shape, dt)
        ks = vs = None
        if dt == V.DT_I8:
            ks, vs = self.state(shape[:3], "f32"), self.state(shape[:3], "f32")
        return PagedCache(k, v, ks, vs)

    def paged_batch(self, seqs: int, max_pages: int) -> PagedBatch:
        """i32 inputs that describe the rows of a step, in this order: cu [seqs + 1],
        lens [seqs], table [seqs, max_pages] (see ``PagedBatch``).  They are read on
        the device, so one program serves every batch of the same shape: unused
        sequences have no rows, and rows past cu[seqs] belong to no sequence."""
        if seqs < 1 or max_pages < 1 or seqs * max_pages >= 1 << 31:
            raise GraphError("paged_batch: at least one sequence and page")
        return PagedBatch(self.input((seqs + 1,), "i32"), self.input((seqs,), "i32"),
                          self.input((seqs, max_pages), "i32"))

    def _paged(self, what, cache, batch, T, Hq, a, b, scale=0.0, window=0):
        """Descriptor words of a paged cache op (vm_abi.h ``PD_*``) with its operands'
        strides, and the buffers of the cache and the batch that follow it."""
        N, Hkv, P, hd = cache.dims
        B, MP = batch.table.shape
        if batch.cu.shape != (B + 1,) or batch.lens.shape != (B,):
            raise GraphError(f"{what}: cu is [seqs + 1] and lens [seqs] of the table's seqs")
        for t in (batch.cu, batch.lens, batch.table):
            if t.dtype != V.DT_I32 or t.view:
                raise GraphError(f"{what}: cu, lens and table are i32")
        if MP * P >= 1 << 31:
            raise GraphError(f"{what}: positions of a sequence fit 31 bits")
        ks = cache.k_scale.buf if cache.k_scale is not None else cache.k.buf
        vs = cache.v_scale.buf if cache.v_scale is not None else cache.v.buf
        return [T, Hq, Hkv, hd, P, N, B, MP, cache.k.dtype, *a, *b, V.f32_bits(scale), window] + [0] * 8, \
            [ks, vs, batch.cu.buf, batch.lens.buf, batch.table.buf]

    def cache_append(self, cache: PagedCache, batch: PagedBatch, k: Tensor, v: Tensor) -> None:
        """Write the new rows' keys and values, [T, heads, head_dim] (tensors or views
        of wider rows), into the cache's pages in place: row r of sequence s is
        position lens[s] - (cu[s + 1] - r).  Pages of i8 take rint(x / scale) of each
        row's scale = max|x| / 127, both f32 (a row of zeros: scale 0; one with an
        infinity or NaN: scale NaN).  Not written: rows of no sequence, sequences whose
        length is less than their new rows or more than the table's pages hold, and
        positions whose table entry is no page (any number outside [0, N)).  Two
        sequences' new rows must not share a position of a page."""
        what = "cache_append"
        dt = self._floats(what, k, v)
        if k.shape != v.shape or len(k.shape) != 3 or k.shape[1:] != (cache.dims[1], cache.dims[3]):
            raise GraphError(f"{what}: k and v are [rows, {cache.dims[1]}, {cache.dims[3]}], not {k.shape} and {v.shape}")
        if cache.k.dtype not in (dt, V.DT_I8):
            raise GraphError(f"{what}: rows of {V.DT_NAMES[dt]} into pages of {V.DT_NAMES[cache.k.dtype]}")
        if k.shape[0] < 1:
            raise GraphError(f"{what}: no rows")
        (kb, *ka), (vb, *va) = self._heads_view(k, what), self._heads_view(v, what)
        words, bufs = self._paged(what, cache, batch, k.shape[0], cache.dims[1], ka, va)
        desc = self.add_aux(words + [cache.v.buf] + bufs)
        self.emit(V.Instr(V.OP_CACHE_APPEND, dst=cache.k.buf, a=kb, b=vb, n=k.shape[0], aux=desc))

    def cache_read(self, cache: PagedCache, batch: PagedBatch, rows: int, dtype="f32") -> tuple:
        """The keys and values that ``cache_append`` of the same batch has its rows
        at, as two tensors [rows, heads, head_dim]: with cu the sums of lens, whole
        sequences one after another.  i8 pages give q * scale, rounded once to
        ``dtype``.  Rows that append would not write are 0."""
        what = "cache_read"
        dt = _dt(dtype)
        if dt not in (V.DT_F32, V.DT_F16, V.DT_BF16) or rows < 1:
            raise GraphError(f"{what}: at least one row of f32, f16 or bf16")
        N, Hkv, P, hd = cache.dims
        words, bufs = self._paged(what, cache, batch, rows, Hkv, (0, 0, 0), (0, 0, 0))
        k, v = self._new((rows, Hkv, hd), dt), self._new((rows, Hkv, hd), dt)
        desc = self.add_aux(words + [v.buf] + bufs)
        self.emit(V.Instr(V.OP_CACHE_READ, dst=k.buf, a=cache.k.buf, b=cache.v.buf, n=rows, aux=desc))
        return k, v

    def paged_attention(self, q: Tensor, cache: PagedCache, batch: PagedBatch, scale: float,
                        window: int = 0) -> Tensor:
        """Causal attention of the new rows' queries q [T, Hq, head_dim] (a tensor or a
        view of wider rows) over the cache, their own positions included (``cache_append``
        first): the row at position p of a sequence sees positions p' <= p, with
        ``window`` > 0 only those above p - window, and query head h reads kv head
        h // (Hq // heads).  Chunks and single tokens mix freely in one batch.
        Positions whose table entry is no page are not seen.  Rows that see nothing,
        rows of no sequence and rows of a sequence whose length is less than its
        new rows or more than its pages hold are 0.  Sums and softmax are f32.
        Returns [T, Hq, head_dim] of q's dtype, which is the pages' or any for i8."""
        what = "paged_attention"
        dt = self._floats(what, q)
        N, Hkv, P, hd = cache.dims
        buf, rs, hs, off = self._heads_view(q, what)
        T, Hq, qd = q.shape
        if qd != hd or Hq < 1 or Hq % Hkv or Hq // Hkv > V.PAGED_MAX_GROUP or T < 1:
            raise GraphError(f"{what}: queries {q.shape} of {Hkv} kv heads of {hd} (at most {V.PAGED_MAX_GROUP} to one)")
        if cache.k.dtype not in (dt, V.DT_I8):
            raise GraphError(f"{what}: queries of {V.DT_NAMES[dt]} over pages of {V.DT_NAMES[cache.k.dtype]}")
        if not (scale > 0 and math.isfinite(scale)) or window < 0 or window >= 1 << 31:
            raise GraphError(f"{what}: scale > 0 and window >= 0")
        words, bufs = self._paged(what, cache, batch, T, Hq, (rs, hs, off), (0, 0, 0), scale, window)
        dst = self._new(q.shape, dt)
        desc = self.add_aux(words + [cache.v.buf] + bufs)
        self.emit(V.Instr(V.OP_PAGED_ATTN, dst=dst.buf, a=buf, b=cache.k.buf, n=T, imm=Hq, aux=desc))
        return dst

    # ---- dynamic slices / gathers ------------------------------------------------
    def dynamic_slice(self, a: Tensor, starts, sizes) -> Tensor:
        a = self.materialize(a)
        rank = len(a.shape)
        st = _row_major_strides(a.shape)
        clamp = [a.shape[d] - sizes[d] for d in range(rank)]
        ids = [s.buf for s in starts]
        is64 = int(starts[0].dtype == V.DT_I64) if starts else 0
        off = self.add_aux([rank] + list(sizes) + st + clamp + [0] * rank + ids + [is64])
        dst = self._new(sizes, a.dtype)
        self.emit(V.Instr(V.OP_DYNAMIC_SLICE, dst=dst.buf, a=a.buf, n=dst.n,
                          aux=off, reads_hint=tuple(ids)))
        return dst

    def dynamic_update_slice(self, dst: Tensor, upd: Tensor, starts) -> None:
        """In place: dst[starts ...] = upd (the loop-carry form)."""
        upd = self.materialize(upd)
        rank = len(dst.shape)
        st = _row_major_strides(dst.shape)
        clamp = [dst.shape[d] - upd.shape[d] for d in range(rank)]
        ids = [s.buf for s in starts]
        is64 = int(starts[0].dtype == V.DT_I64) if starts else 0
        off = self.add_aux([rank] + list(upd.shape) + st + clamp + [0] * rank + ids + [is64])
        self.emit(V.Instr(V.OP_DYNAMIC_UPDATE_SLICE, dst=dst.buf, a=upd.buf,
                          n=upd.n, aux=off, reads_hint=tuple(ids)))

    def take_rows(self, table: Tensor, idx: Tensor) -> Tensor:
        """out[i, :] = table[clamp(idx[i]), :] (embedding lookup as a
        stablehlo.gather with one index component)."""
        table, idx = self.materialize(table), self.materialize(idx)
        rows, width = table.shape
        nidx = 1
        out_shape = tuple(idx.shape) + (width,)
        out_rank = len(out_shape)
        op_stride = [0] * (out_rank - 1) + [1]
        si_stride = _row_major_strides(idx.shape) + [0]
        words = [out_rank, nidx, 0, int(idx.dtype == V.DT_I64), 0, idx.buf]
        words += list(out_shape) + op_stride + si_stride + [width] + [rows - 1]
        off = self.add_aux(words)
        dst = self._new(out_shape, table.dtype)
        self.emit(V.Instr(V.OP_GATHER_INDEX, dst=dst.buf, a=table.buf, n=dst.n,
                          aux=off, reads_hint=(idx.buf,)))
        return dst

    def copy_into(self, dst: Tensor, src: Tensor) -> None:
        """dst <- src (elementwise copy; used for loop-carry updates)."""
        src = self.materialize(src)
        op = V.OP_COPY_F32 if src.dtype == V.DT_F32 else V.OP_CONVERT
        self.emit(V.Instr(op, dst=dst.buf, a=src.buf, n=src.n))

    # ---- control flow --------------------------------------------------------------
    def begin(self) -> None:
        self._stack.append([])

    def end(self) -> list:
        return self._stack.pop()

    def for_loop(self, trips: int, body: list) -> None:
        self.emit(V.Instr(V.OP_FOR, b=trips, n=0, imm=0))
        self._pending_region(self._last_list()[-1], [], body)

    def while_loop(self, cond: Tensor, cond_list: list, body: list) -> None:
        self.emit(V.Instr(V.OP_WHILE, dst=cond.buf))
        self._pending_region(self._last_list()[-1], cond_list, body)

    def if_(self, flag: Tensor, then_list: list, else_list: list) -> None:
        self.emit(V.Instr(V.OP_IF, dst=flag.buf))
        self._pending_region(self._last_list()[-1], then_list, else_list)

    def _last_list(self) -> list:
        return self._stack[-1] if self._stack else self.instrs

    def _pending_region(self, ins, first, second) -> None:
        self.regions.append((ins, first, second))

    # ---- build ----------------------------------------------------------------------
    def build(self) -> V.VMProgram:
        # Region sub-lists are appended after the root list; a region nested in
        # another's sub-list gets its ranges fixed the same way (BFS order).
        instrs = list(self.instrs)
        main_len = len(instrs)
        pending = list(self.regions)
        placed = set()
        while pending:
            progress = False
            for item in list(pending):
                ins, first, second = item
                if not any(ins is x for x in instrs):
                    continue
                pending.remove(item)
                progress = True
                a = len(instrs)
                instrs.extend(first)
                n = len(instrs)
                instrs.extend(second)
                if ins.op == V.OP_FOR:
                    ins.n, ins.imm = n, len(second)
                else:
                    ins.a, ins.b, ins.n, ins.imm = a, len(first), n, len(second)
                placed.add(id(ins))
            if not progress:
                raise GraphError("region instruction not reachable from root")
        bufs, off = [], 0
        for i, (n, dt) in enumerate(self.buffers):
            size = n * V.DT_SIZE[dt]
            if i in self.states:            # takes no arena bytes: placed past them below
                bufs.append(V.Buffer(0, size, dt, True))
                continue
            if i in self.aliases:           # shares its parent's memory
                parent, byte_off = self.aliases[i]
                bufs.append(V.Buffer(bufs[parent].arena_byte_offset + byte_off, size, dt))
                continue
            bufs.append(V.Buffer(off, size, dt))
            off += max(ARENA_SLOT, -(-size // V.ARENA_ALIGN) * V.ARENA_ALIGN)
        V.place_states(bufs, off)
        return V.VMProgram(
            arena_bytes=off, buffers=bufs,
            inputs=[t.buf for t in self.inputs],
            outputs=[t.buf for t in self.outputs],
            input_shapes=[t.shape for t in self.inputs],
            output_shapes=[t.shape for t in self.outputs],
            consts=list(self.consts), instrs=instrs, main_len=main_len,
            aux=list(self.aux))


ARENA_SLOT = 64


def rotary_grad_workers(T: int, H: int) -> int:
    """Tiles of a rotary gradient, each with a partial sum of dweight of its own: one per
    16 (row, head) pairs up to 256, a CU's worth each."""
    return max(1, min(256, T * H // 16))
