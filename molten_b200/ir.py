"""Dataflow IR: the graph a user builds and the fusion engine partitions.

Drop-in for the reference's ``molten/ir.py``: the same ``OpType`` members in
the same order (``molten/ir.py:20-66``), the same ``TensorShape``/``Op``
fields (``ir.py:69-103``) and the same ``DataflowGraph`` builders and analysis
methods (``ir.py:106-236``).  Additions, all optional keyword arguments or new
helpers so that reference callers are unaffected:

* ``rms_norm(..., eps=1e-6)`` records ``eps`` on the RMS op (the reference
  hard-codes 1e-6 in its kernels, ``codegen.py:286``).
* ``clamp(x, lo, hi)`` stores the bounds in ``attrs["min"]``/``attrs["max"]``
  (the reference has a CLAMP op type but no semantics for it).
* ``causal_mask(period, offset)`` adds a CONSTANT whose value is generated
  from indices: 0 where ``col <= (row mod period) + offset``, ``-inf`` above.
* small builders for the remaining unary ops (``gelu``, ``silu`` ...).
* ``ModelOpType``: the operators of a decode step (4-bit products, rotary
  positions on several axes, window attention, sampling), which the reference
  does not have.  They are an enum of their own because the members of
  ``OpType`` and their values are the reference's interface.
"""

from __future__ import annotations

from dataclasses import dataclass, field
from enum import Enum, auto
from typing import Optional


class OpType(Enum):
    # elementwise
    ADD = auto()
    SUB = auto()
    MUL = auto()
    DIV = auto()
    NEG = auto()
    SQRT = auto()
    RSQRT = auto()
    EXP = auto()
    LOG = auto()
    TANH = auto()
    SIGMOID = auto()
    GELU = auto()
    SILU = auto()
    RELU = auto()
    ABS = auto()
    CLAMP = auto()
    # row reductions
    SUM = auto()
    MEAN = auto()
    MAX = auto()
    MIN = auto()
    NORM = auto()
    RMS = auto()
    # contractions
    MATMUL = auto()
    DOT = auto()
    OUTER = auto()
    # attention primitives
    SOFTMAX = auto()
    ROTATE = auto()
    # data movement
    TRANSPOSE = auto()
    RESHAPE = auto()
    SLICE = auto()
    CONCAT = auto()
    BROADCAST = auto()
    # graph boundary
    INPUT = auto()
    OUTPUT = auto()
    CONSTANT = auto()


class ModelOpType(Enum):
    """Operators beyond the reference's (``molten_b200/decode.py``)."""
    MATVEC_Q4 = auto()
    ROTATE_POSITIONS = auto()
    WINDOW_ATTENTION = auto()
    SAMPLE = auto()


ELEMENTWISE_OPS = frozenset({
    OpType.ADD, OpType.SUB, OpType.MUL, OpType.DIV,
    OpType.NEG, OpType.SQRT, OpType.RSQRT, OpType.EXP,
    OpType.LOG, OpType.TANH, OpType.SIGMOID, OpType.GELU,
    OpType.SILU, OpType.RELU, OpType.ABS, OpType.CLAMP,
})

REDUCTION_OPS = frozenset({
    OpType.SUM, OpType.MEAN, OpType.MAX, OpType.MIN,
    OpType.NORM, OpType.RMS, OpType.SOFTMAX,
})

BOUNDARY_OPS = frozenset({OpType.INPUT, OpType.OUTPUT, OpType.CONSTANT})


@dataclass
class TensorShape:
    """Shape with optional symbolic (string) dimensions."""
    dims: list

    def __repr__(self):
        return "(" + ", ".join(str(d) for d in self.dims) + ")"

    @property
    def ndim(self) -> int:
        return len(self.dims)

    @property
    def is_fully_known(self) -> bool:
        return all(isinstance(d, int) for d in self.dims)


@dataclass
class Op:
    """One node of the dataflow graph."""
    id: int
    op_type: OpType
    name: str = ""
    inputs: list = field(default_factory=list)
    shape: Optional[TensorShape] = None
    dtype: str = "float16"
    attrs: dict = field(default_factory=dict)
    fusable: bool = True
    memory_bound: bool = False
    reduction_dim: Optional[int] = None

    def __repr__(self):
        return f"Op({self.id}: {self.op_type.name} '{self.name}' {self.shape})"


class DataflowGraph:
    """A DAG of ``Op`` nodes keyed by integer id (ids are insertion order)."""

    def __init__(self, name: str = "unnamed"):
        self.name = name
        self.ops: dict[int, Op] = {}
        self._next_id = 0
        self._outputs: list[int] = []

    # ------------------------------------------------------------------ build
    def add_op(self, op_type: OpType, inputs: list = None, name: str = "",
               shape: Optional[TensorShape] = None, dtype: str = "float16",
               **attrs) -> int:
        op_id = self._next_id
        self._next_id += 1
        self.ops[op_id] = Op(id=op_id, op_type=op_type, name=name,
                             inputs=list(inputs or []), shape=shape,
                             dtype=dtype, attrs=attrs)
        return op_id

    def add_input(self, name: str, shape: TensorShape,
                  dtype: str = "float16") -> int:
        return self.add_op(OpType.INPUT, name=name, shape=shape, dtype=dtype)

    def add_output(self, input_id: int, name: str = "output") -> int:
        out_id = self.add_op(OpType.OUTPUT, [input_id], name=name,
                             shape=self.ops[input_id].shape)
        self._outputs.append(out_id)
        return out_id

    def add_constant(self, name: str, value: float) -> int:
        return self.add_op(OpType.CONSTANT, name=name, value=value)

    # ------------------------------------------------------------- builders
    def add(self, a: int, b: int, name: str = "") -> int:
        return self.add_op(OpType.ADD, [a, b], name)

    def sub(self, a: int, b: int, name: str = "") -> int:
        return self.add_op(OpType.SUB, [a, b], name)

    def mul(self, a: int, b: int, name: str = "") -> int:
        return self.add_op(OpType.MUL, [a, b], name)

    def div(self, a: int, b: int, name: str = "") -> int:
        return self.add_op(OpType.DIV, [a, b], name)

    def matmul(self, a: int, b: int, name: str = "") -> int:
        return self.add_op(OpType.MATMUL, [a, b], name)

    def softmax(self, x: int, dim: int = -1, name: str = "") -> int:
        op_id = self.add_op(OpType.SOFTMAX, [x], name)
        self.ops[op_id].reduction_dim = dim
        return op_id

    def rms_norm(self, x: int, weight: int, name: str = "",
                 eps: float = 1e-6) -> int:
        """x / rms(x) * weight, expanded to RMS -> DIV -> MUL."""
        rms_id = self.add_op(OpType.RMS, [x], f"{name}_rms", eps=eps)
        div_id = self.div(x, rms_id, f"{name}_div")
        return self.mul(div_id, weight, f"{name}_scale")

    def rope(self, x: int, freqs: int, name: str = "", sin: Optional[int] = None,
             style: Optional[str] = None, positions: Optional[int] = None,
             sections: Optional[list] = None) -> int:
        """ROTATE: rotary position embedding of x [..., seq, heads, head_dim].

        ``rope(x, freqs)`` is the reference's builder (``ir.py:175-176``);
        its table layout is not specified there, so here ``freqs`` is
        [seq, head_dim] holding each pair's (cos, sin) interleaved.  With
        ``sin`` given, ``freqs`` is the cos table and both are
        [seq, head_dim/2] -- the form of ``benchmarks/ops.py:24-35``.
        ``style``: "interleaved" pairs (2i, 2i+1) as in ops.py (default) or
        "half" pairs (i, i + head_dim/2).  The result has x's dtype.

        ``positions`` (int32, [axes, ..., seq], or [..., seq] for one axis)
        gives every token's row of the table instead of its own index; the
        tables may then have any number of rows.  With several axes (time,
        height, width ...) ``sections`` counts the pairs each axis turns, in
        order (they sum to head_dim/2; at most 4).  A negative position marks
        padding, whose pairs are left as they are; a position past the table
        sets a bit of the status word and leaves them too."""
        inputs = [x, freqs] + ([sin] if sin is not None else [])
        attrs = {"style": style} if style else {}
        if positions is not None:
            attrs["sections"] = [int(v) for v in sections] if sections is not None else None
            attrs["packed"] = sin is None
            return self.add_op(ModelOpType.ROTATE_POSITIONS, inputs + [positions], name, **attrs)
        if sections is not None:
            raise ValueError("rope: sections need positions")
        return self.add_op(OpType.ROTATE, inputs, name, **attrs)

    def matvec_q4(self, x: int, qweight: int, scales: int, zeros: Optional[int] = None,
                  name: str = "") -> int:
        """x [..., K] times 4-bit weights: y[..., n] = sum_k x[..., k]
        (q[n, k] - zeros[n, k // G]) * scales[n, k // G].

        ``qweight`` is uint8 [N, K/2], the even k in the low nibble;
        ``scales`` and ``zeros`` are [N, K/G] floats with G = 32, 64 or 128;
        without ``zeros`` the zero point is 8.  At most 32 rows of x; the
        result has x's dtype."""
        return self.add_op(ModelOpType.MATVEC_Q4,
                           [x, qweight, scales] + ([zeros] if zeros is not None else []), name)

    def window_attention(self, q: int, k: int, v: int, lengths: Optional[int] = None,
                         window: Optional[int] = None, sinks: int = 0,
                         scale: Optional[float] = None, name: str = "") -> int:
        """Causal attention over a sliding window and the first ``sinks``
        keys: q [batch, new, heads, d], k and v [batch, cache, kv_heads, d]
        (heads a multiple of kv_heads; bf16 or fp16, d <= 128).

        ``lengths`` (int32 [batch], default ``cache``) counts each request's
        valid keys, its new tokens the last of them: query i stands at
        p = length - new + i and sees key j iff j <= p, j < length and
        (j > p - window or j < sinks).  ``window=None``: every earlier key.
        A query that sees no key gets zeros.  ``scale`` defaults to
        1/sqrt(d).  Keys that no query sees are never used, whatever they
        hold."""
        return self.add_op(ModelOpType.WINDOW_ATTENTION,
                           [q, k, v] + ([lengths] if lengths is not None else []), name,
                           window=None if window is None else int(window), sinks=int(sinks),
                           scale=None if scale is None else float(scale))

    def sample(self, logits: int, u: int, temperature: Optional[int] = None,
               top_k: Optional[int] = None, top_p: Optional[int] = None,
               min_p: Optional[int] = None, name: str = "") -> int:
        """One token per row of logits [..., V] (int32 [...]), drawn with the
        given random numbers u in [0, 1).

        Every parameter is a vector with one value per row (float32; top_k
        int32) or a scalar constant.  In order: w = exp((x - max) /
        temperature); keep the ``top_k`` largest (<= 0: all); of those the
        smallest set of largest ones whose weight is at least ``top_p`` of
        theirs (>= 1: all); of those the ones with w >= ``min_p`` (the largest
        w is 1).  Equal logits count by index, the lowest first.  The token is
        the first, by index, at which the running weight of the kept tokens
        exceeds u times their sum.  ``temperature`` below 1e-30 takes the
        largest logit.  NaN logits and -inf are never drawn (a row of nothing
        else gives -1); +inf counts as the largest finite number of its
        type.  Weights and sums have 64 bits."""
        params = {"temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p}
        given = [k for k, v in params.items() if v is not None]
        return self.add_op(ModelOpType.SAMPLE, [logits, u] + [params[k] for k in given], name,
                           params=given)

    def transpose(self, x: int, name: str = "") -> int:
        """TRANSPOSE of the last two dims (a matrix [N, K] -> [K, N]).  As
        a MATMUL's B operand it costs nothing: the GEMM reads the original
        rows K-major."""
        return self.add_op(OpType.TRANSPOSE, [x], name)

    def unary(self, op_type: OpType, x: int, name: str = "", **attrs) -> int:
        return self.add_op(op_type, [x], name, **attrs)

    def gelu(self, x: int, name: str = "") -> int:
        return self.unary(OpType.GELU, x, name)

    def silu(self, x: int, name: str = "") -> int:
        return self.unary(OpType.SILU, x, name)

    def sigmoid(self, x: int, name: str = "") -> int:
        return self.unary(OpType.SIGMOID, x, name)

    def relu(self, x: int, name: str = "") -> int:
        return self.unary(OpType.RELU, x, name)

    def exp(self, x: int, name: str = "") -> int:
        return self.unary(OpType.EXP, x, name)

    def clamp(self, x: int, lo: Optional[float] = None,
              hi: Optional[float] = None, name: str = "") -> int:
        return self.add_op(OpType.CLAMP, [x], name, min=lo, max=hi)

    def causal_mask(self, period: Optional[int] = None, offset: int = 0,
                    name: str = "causal_mask") -> int:
        """Index-generated additive mask: 0 on/below the diagonal, -inf above.

        Element (row, col) of the mask is ``-inf`` iff
        ``col > (row mod period) + offset``; ``period=None`` means the number
        of columns of the tensor it is added to.
        """
        return self.add_op(OpType.CONSTANT, name=name, kind="causal_mask",
                           period=period, offset=offset, value=None)

    # -------------------------------------------------------------- analysis
    def inputs(self) -> list:
        return [op for op in self.ops.values() if op.op_type == OpType.INPUT]

    def outputs(self) -> list:
        return [op for op in self.ops.values() if op.op_type == OpType.OUTPUT]

    def consumers(self, op_id: int) -> list:
        return [oid for oid, op in self.ops.items() if op_id in op.inputs]

    def producers(self, op_id: int) -> list:
        return self.ops[op_id].inputs

    def topological_order(self) -> list:
        """Depth-first post-order over op ids, visiting roots by id."""
        seen: set = set()
        order: list = []
        for root in self.ops:
            if root in seen:
                continue
            # iterative DFS so that deep chains do not hit the recursion limit
            stack = [(root, 0)]
            seen.add(root)
            while stack:
                node, i = stack[-1]
                ins = self.ops[node].inputs
                if i < len(ins):
                    stack[-1] = (node, i + 1)
                    nxt = ins[i]
                    if nxt not in seen:
                        seen.add(nxt)
                        stack.append((nxt, 0))
                else:
                    stack.pop()
                    order.append(node)
        return order

    def is_elementwise(self, op_id: int) -> bool:
        return self.ops[op_id].op_type in ELEMENTWISE_OPS

    def is_reduction(self, op_id: int) -> bool:
        return self.ops[op_id].op_type in REDUCTION_OPS

    def __repr__(self):
        lines = [f"DataflowGraph '{self.name}' ({len(self.ops)} ops):"]
        lines += [f"  {self.ops[i]}" for i in self.topological_order()]
        return "\n".join(lines)
