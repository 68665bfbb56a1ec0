"""Parameter blocks and launches of the model operators (``decode.py``).

Every call reads pointers and strides from the tensors it is given; nothing is
kept from one call for the next but what the shapes decide (the sizes' part of
the parameter block, the launch geometry).  Workspaces come from torch's
allocator on the launching stream, one per call, so calls on several streams
and captured graphs never share one.

A call has two ways in.  ``launch_model_op`` runs a model operator among the
sub-kernels of any plan and brings operands into a layout the kernel takes.
``short_call`` is the short way for a graph that is one model operator, called
with the declared shapes or again with those of its last call: single tokens run
for a few microseconds, less than the general path's bookkeeping.  It declines
(``NotImplemented``) whatever is not plain, and the general path takes over.
Its steps are native (``csrc/call.cpp``) where that library is built, 4 to 6 us a
call, else ``ModelCall``'s, 9 to 11.
"""

from __future__ import annotations

import ctypes
import math
from struct import Struct

from . import _capi
from .decode import SAMPLE_PARAMS, SMS
from .ir import ModelOpType
from .lowering import DTYPE_SIZE

LOG2E = math.log2(math.e)


def _merged(t, keep: int):
    """t with its leading dims merged into one and its last ``keep`` dims as
    they are, without a copy where the strides allow it and the last dim is
    contiguous; else a contiguous copy."""
    tail = tuple(t.shape[t.dim() - keep:])
    lead = 1
    for d in t.shape[:t.dim() - keep]:
        lead *= d
    if t.stride(-1) == 1 or t.shape[-1] == 1:
        try:
            return t.view((lead,) + tail)
        except RuntimeError:
            pass
    return t.contiguous().view((lead,) + tail)


def _copied(t):
    """t in memory of its own, contiguous and aligned."""
    return t.clone() if t.is_contiguous() else t.contiguous()


def _aligned(t, nbytes: int, strides) -> bool:
    return t.data_ptr() % nbytes == 0 and all(s * t.element_size() % nbytes == 0 for s in strides)


class _Bound:
    """One model sub-kernel on one device: its module, launch geometry and the
    part of its parameter block that the shapes decide."""

    def __init__(self, spec, i: int, device: int):
        self.sk = spec.plan.kernels[i]
        self.c = self.sk.config
        self.entry = spec.entries[i]
        self.module = spec.module(device)
        self.device = device
        self.setup()

    def config(self, grid, block: int, cluster: int = 1, smem: int = 0):
        from .runtime import PDL
        cfg = _capi.LaunchCfg()
        cfg.grid[:] = [grid, 1, 1]
        cfg.block[:] = [block, 1, 1]
        cfg.cluster[:] = [cluster, 1, 1]
        cfg.smem_bytes = smem
        cfg.flags = _capi.LAUNCH_PDL if PDL else 0
        return ctypes.byref(cfg), cfg

    def tail(self, args_type, first: str) -> bytes:
        """The static end of a parameter block, from field ``first`` on, with
        this kernel's sizes."""
        a = args_type()
        self.fill(a)
        return bytes(a)[getattr(args_type, first).offset:]

    def launch(self, block: bytes, stream: int, cfg=None, entry=None) -> None:
        entry = entry or self.entry
        rc = self.module.lib.molten_launch(self.module.handle, entry, cfg or self.cfg[0], block,
                                           len(block), stream)
        if rc:
            raise _capi.MoltenError(f"launching {entry.decode()} failed (code {rc}): "
                                    f"{_capi.last_error()}")

    def need_aligned(self, j: int, t, nbytes: int) -> None:
        if t.data_ptr() % nbytes:
            name = next(o.name for o in self.sk.operands if o.index == j) if j >= 0 else "output"
            raise _capi.MoltenError(f"{'input ' + repr(name) if j >= 0 else name} at "
                                    f"{t.data_ptr():#x} is not {nbytes}-byte aligned as kernel "
                                    f"{self.entry.decode()} requires")

    # per operator: setup(); fill(args); conform(ins) -> ins the kernel takes;
    # run(ins, out, stream) on such ins; short() -> (parameter block for
    # contiguous operands, (offset, operand or -1 for the output) of each pointer
    # in it, tensor maps), or None

    def short(self):
        return None


class _Q4(_Bound):
    head = Struct("<5Qq")

    def setup(self):
        c = self.c
        self.cfg = self.config(c["teams"] * c["ksplit"], c["block"], c["ksplit"], c["smem"])
        self.rest = self.tail(_capi.Q4Args, "n")

    def fill(self, a):
        c = self.c
        a.n, a.m, a.k = c["n"], c["m"], c["k"]
        a.warps_n_log, a.ksplit_log = c["warps_n"].bit_length() - 1, c["ksplit"].bit_length() - 1
        a.chunk, a.tiles, a.teams = c["chunk"], c["tiles"], c["teams"]

    def conform(self, ins):
        x = _merged(ins[0], 1)
        if not _aligned(x, 16, x.stride()[:-1] if x.shape[0] > 1 else ()):
            x = _copied(x)
        self.need_aligned(1, ins[1], 16)
        for j in range(2, len(ins)):
            self.need_aligned(j, ins[j], ins[j].element_size())
        return [x] + ins[1:]

    def short(self):
        n = len(self.sk.operands)
        return (self.head.pack(0, 0, 0, 0, 0, self.c["k"]) + self.rest,
                [(8 * j, j) for j in range(n)] + [(32, -1)], [])

    def run(self, ins, out, stream):
        x = ins[0]
        block = self.head.pack(x.data_ptr(), ins[1].data_ptr(), ins[2].data_ptr(),
                               ins[3].data_ptr() if len(ins) > 3 else 0, out.data_ptr(),
                               x.stride(-2) if x.dim() > 1 else self.c["k"])
        self.launch(block + self.rest, stream)


class _Rope(_Bound):
    head = Struct("<6Q4q")

    def setup(self):
        c = self.c
        self.cfg = self.config(-(-c["tokens"] // c["tokens_per_cta"]), c["block"])
        self.rest = self.tail(_capi.RopePosArgs, "heads")
        self.status = _capi.status_word(self.device)

    def fill(self, a):
        c = self.c
        a.heads, a.dim = c["heads"], c["dim"]
        a.axes, a.head_lanes, a.tokens_per_cta = len(c["sections"]), c["head_lanes"], c["tokens_per_cta"]
        end = 0
        for j, width in enumerate(c["sections"]):
            end += width
            a.bound[j] = end

    def conform(self, ins):
        c = self.c
        x = _merged(ins[0], 2)
        if c["xvec"]:
            slot = min(16, c["vec"] * x.element_size())
            if not _aligned(x, slot, x.stride()[:-1]):
                x = _copied(x)
        if c["tvec"]:
            for j in range(1, len(ins) - 1):
                self.need_aligned(j, ins[j], c["table_slot"])
        return [x] + ins[1:]

    def short(self):
        c, n = self.c, len(self.sk.operands)
        return (self.head.pack(0, 0, 0, 0, 0, self.status, c["tokens"], c["heads"] * c["dim"], c["dim"],
                               c["table_rows"]) + self.rest,
                [(0, 0), (8, 1), (16, n - 2), (24, n - 1), (32, -1)], [])

    def run(self, ins, out, stream):
        c, x = self.c, ins[0]
        if c["xvec"]:
            self.need_aligned(-1, out, min(16, c["vec"] * out.element_size()))
        block = self.head.pack(x.data_ptr(), ins[1].data_ptr(), ins[-2].data_ptr(),
                               ins[-1].data_ptr(), out.data_ptr(), self.status,
                               c["tokens"], x.stride(-3), x.stride(-2), c["table_rows"])
        self.launch(block + self.rest, stream)


class _Window(_Bound):
    head = Struct("<6Q9q")
    tiles_head = Struct("<4Q3q")
    dims, strides, box = Struct("<4Q"), Struct("<3Q"), Struct("<4I")

    def setup(self):
        c = self.c
        if c["kind"] == "tiles":
            self.cfg = self.config(min(c["items"] * c["parts"], SMS), c["block"], 1, c["smem"])
            self.rest = self.tail(_capi.WindowTcArgs, "batch")
            self.part = c["items"] * 256 * c["parts"] * (c["dim"] + 4) if c["parts"] > 1 else 0
            self.part_at = _capi.WindowTcArgs.part.offset - _capi.WindowTcArgs.batch.offset
            self.join = self.config(c["items"] * 32, 256)
            self.status = _capi.status_word(self.device)
            self.code = _capi.DT_BF16 if self.sk.operands[0].dtype == "bfloat16" else _capi.DT_F16
        else:
            self.cfg = self.config(c["items"] * c["parts"] * c["ranks"], c["block"], c["ranks"],
                                   c["smem_launch"])
            self.rest = self.tail(_capi.WindowArgs, "batch")
            self.part = c["items"] * c["parts"] * c["rows"] * (c["dim"] + 2) if c["parts"] > 1 else 0
            self.join = self.config(-(-c["items"] * c["rows"] // 4), 128)

    def fill(self, a):
        c = self.c
        a.batch, a.nq, a.cache, a.kv_heads = c["batch"], c["new"], c["cache"], c["kv_heads"]
        a.per, a.dim, a.window, a.sinks = c["per"], c["dim"], c["window"], c["sinks"]
        a.scale_log2 = c["scale"] * LOG2E
        if c["kind"] == "tiles":
            a.positions, a.blocks, a.parts = c["positions"], c["blocks"], c["parts"]
        else:
            a.ranks, a.parts = c["ranks"], c["parts"]

    def conform(self, ins):
        out = list(ins)
        for j in range(3):
            t = ins[j]
            # 16-byte rows: the last dim contiguous, every other stride a
            # multiple of 8 elements (and not 0 where TMA copies the tiles)
            if ((t.stride(3) != 1 and t.shape[3] > 1) or not _aligned(t, 16, t.stride()[:3])
                    or (self.c["kind"] == "tiles"
                        and any(n > 1 and x == 0 for n, x in zip(t.shape, t.stride())))):
                # (a cache that is only misplaced is not copied at every call)
                t = _copied(t) if j == 0 else t.contiguous()
            self.need_aligned(j, t, 16)
            out[j] = t
        return out

    def tensor_maps(self, ins) -> bytes:
        """The TMA descriptors of q, k and v [b, s, h, d], 128 bytes each.  The
        stride of a dim of one element (any number in torch) is replaced by one
        that the encoder takes."""
        c = self.c
        buf = (ctypes.c_char * 448)()
        at = (ctypes.addressof(buf) + 63) & ~63
        encode = self.module.lib.molten_encode_tma_4d
        for n, t in enumerate(ins[:3]):
            b, s, h, d = t.shape
            sb, ss, sh, _ = t.stride()
            box = (64, c["per"], c["positions"], 1) if n == 0 else (64, 1, 128, 1)
            _capi.check(encode(at + 128 * n, self.code, t.data_ptr(), self.dims.pack(d, h, s, b),
                               self.strides.pack(2 * sh if h > 1 else 16, 2 * ss if s > 1 else 16,
                                                 2 * sb if b > 1 else 16),
                               self.box.pack(*box)), "encoding a TMA descriptor")
        return ctypes.string_at(at, 384)

    def short(self):
        c = self.c
        d, kv, heads = c["dim"], c["kv_heads"], c["kv_heads"] * c["per"]
        q, k = (c["new"] * heads * d, heads * d, d), (c["cache"] * kv * d, kv * d, d)
        lengths = [(0, 3)] if len(self.sk.operands) > 3 else []
        if self.part:
            return None
        if c["kind"] == "tiles":
            maps = [(128 * n, n, self.code, self.dims.pack(d, h, s, c["batch"]),
                     self.strides.pack(2 * st[2], 2 * st[1], 2 * st[0]), self.box.pack(*box))
                    for n, (h, s, st, box) in enumerate(
                        [(heads, c["new"], q, (64, c["per"], c["positions"], 1))]
                        + 2 * [(kv, c["cache"], k, (64, 1, 128, 1))])]
            return (bytes(384) + self.tiles_head.pack(0, 0, 0, self.status, *k) + self.rest,
                    [(384, 2)] + [(392 + at, j) for at, j in lengths] + [(400, -1)], maps)
        return (self.head.pack(0, 0, 0, 0, 0, 0, *q, *k, *k) + self.rest,
                [(0, 0), (8, 1), (16, 2)] + [(24 + at, j) for at, j in lengths] + [(32, -1)], [])

    def run(self, ins, out, stream):
        q, k, v = ins[:3]
        lengths = ins[3].data_ptr() if len(ins) > 3 else 0
        c = self.c
        self.need_aligned(-1, out, 16)
        part = None
        if self.part:
            import torch
            part = torch.empty(self.part, dtype=torch.float32, device=q.device)
        if c["kind"] == "tiles":
            block = (self.tensor_maps(ins)
                     + self.tiles_head.pack(v.data_ptr(), lengths, out.data_ptr(), self.status,
                                            *v.stride()[:3]))
            rest = self.rest
            if part is not None:
                rest = (rest[:self.part_at] + part.data_ptr().to_bytes(8, "little")
                        + rest[self.part_at + 8:])
            self.launch(block + rest, stream)
            if part is not None:
                self.launch(block + rest, stream, self.join[0], self.entry + b"_join")
            return
        block = self.head.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), lengths, out.data_ptr(),
                               0 if part is None else part.data_ptr(),
                               *q.stride()[:3], *k.stride()[:3], *v.stride()[:3]) + self.rest
        self.launch(block, stream)
        if part is not None:
            self.launch(block, stream, self.join[0], self.entry + b"_join")


class _Sample(_Bound):
    head = Struct("<7Qq")
    slots = SAMPLE_PARAMS

    def setup(self):
        c = self.c
        self.cfg = self.config(c["rows"] * c["ranks"], c["block"], c["ranks"], c["smem"])
        self.rest = self.tail(_capi.SampleArgs, "rows")
        # where each parameter stands among the tensors of a call
        self.at, n = [], 2
        for name in self.slots:
            given = name in c["params"] and 2 + c["params"].index(name) not in c["scalars"]
            self.at.append(n if given else -1)
            n += given

    def fill(self, a):
        c = self.c
        a.rows, a.vocab, a.run, a.ranks = c["rows"], c["vocab"], c["run"], c["ranks"]
        a.temperature_all, a.top_p_all = 1.0, 1.0        # without a parameter: no limit
        for pos, value in c["scalars"].items():
            name = c["params"][pos - 2]
            # (past 32 bits: every token; below 0: no limit)
            setattr(a, name + "_all", max(-1, min(int(value), 2 ** 31 - 1)) if name == "top_k" else float(value))

    def conform(self, ins):
        x = _merged(ins[0], 1)
        self.need_aligned(0, x, x.element_size())
        return [x] + ins[1:]

    def short(self):
        return (self.head.pack(0, 0, 0, 0, 0, 0, 0, self.c["vocab"]) + self.rest,
                [(0, 0), (8, 1)] + [(16 + 8 * i, j) for i, j in enumerate(self.at) if j > 0] + [(48, -1)], [])

    def run(self, ins, out, stream):
        x = ins[0]
        t, k, p, m = [ins[j].data_ptr() if j > 0 else 0 for j in self.at]
        block = self.head.pack(x.data_ptr(), ins[1].data_ptr(), t, k, p, m, out.data_ptr(),
                               x.stride(-2))
        self.launch(block + self.rest, stream)


_BOUND = {ModelOpType.MATVEC_Q4: _Q4, ModelOpType.ROTATE_POSITIONS: _Rope,
          ModelOpType.WINDOW_ATTENTION: _Window, ModelOpType.SAMPLE: _Sample}

# operands a kernel takes as strided views; the rest are made contiguous
STRIDED = {ModelOpType.MATVEC_Q4: (0,), ModelOpType.ROTATE_POSITIONS: (0,),
           ModelOpType.WINDOW_ATTENTION: (0, 1, 2), ModelOpType.SAMPLE: (0,)}


def _bound(spec, i: int, device: int) -> _Bound:
    key = ("model", i, device)
    b = spec._cfgs.get(key)
    if b is None:
        b = spec._cfgs[key] = _BOUND[spec.plan.kernels[i].config["op"]](spec, i, device)
    return b


def launch_model_op(spec, i: int, env: dict, device: int, stream: int) -> None:
    """Launch sub-kernel ``i`` of ``spec`` on ``stream``."""
    b = _bound(spec, i, device)
    # (operand positions of scalars are left out: SAMPLE's ``at`` counts them)
    ins = [env[o.op_id] for o in b.sk.operands]
    b.run(b.conform(ins), env[b.sk.outputs[0].op_id], stream)


def _extent(t):
    """(first byte, byte behind the last) of a tensor's memory."""
    start = t.data_ptr()
    if t.is_contiguous():
        return start, start + t.nbytes
    if t.numel() == 0:
        return start, start
    return start, start + (1 + sum((d - 1) * s for d, s in zip(t.shape, t.stride()))) * t.element_size()


def _overlap_rules(plan) -> list:
    """What each output may not overlap: [[(place among the inputs, or place
    among the outputs - their number, the input is RoPE's x, name)]]."""
    places = {o: n - len(plan.outputs) for n, o in enumerate(plan.outputs)}
    places.update((o, n) for n, o in enumerate(plan.inputs))
    rules = []
    for n, o in enumerate(plan.outputs):
        found = [(m - len(plan.outputs), False, "another output") for m in range(n)]
        i = next(i for i, sk in enumerate(plan.kernels) if any(w.op_id == o for w in sk.outputs))
        for j, sk in enumerate(plan.kernels[i:], i):
            if "model" not in (sk.family, plan.kernels[i].family):
                continue
            for operand in sk.operands:
                if operand.op_id in places and operand.op_id != o:
                    turned = (j == i and sk.config["op"] == ModelOpType.ROTATE_POSITIONS and operand.index == 0)
                    found.append((places[operand.op_id], turned, f"the input {operand.name!r}"))
        rules.append(found)
    return rules


def refuse_overlap(plan, tensors, outs) -> None:
    """In a plan with a model operator, an output may not lie in memory that
    other blocks of its kernel, or a kernel after it, still read, nor in
    another output's.  (RoPE turns pairs where they are: its x may be its
    output.  Kernels of the other families are left to the caller.)"""
    if plan.overlap is None:
        model = any(sk.family == "model" for sk in plan.kernels)
        plan.overlap = _overlap_rules(plan) if model else []
    every = list(tensors) + list(outs)               # (negative places count from the end)
    extents = [_extent(t) for t in every] if plan.overlap else None
    for n, rules in enumerate(plan.overlap):
        start, end = extents[n - len(outs)]
        for place, turned, name in rules:
            first, last = extents[place]
            if max(start, first) < min(end, last):       # (never with an empty tensor)
                t, out = every[place], outs[n]
                if turned and first == start and t.is_contiguous() and t.dtype == out.dtype:
                    continue
                raise RuntimeError(f"{plan.name}: an output overlaps {name}")


class ModelCall:
    """The short way into a plan that is one model operator: ``call(tensors)``
    with contiguous, 16-byte aligned tensors on the current device, on its
    current stream; ``NotImplemented`` for anything else."""

    def __init__(self, spec, tensors):
        import torch
        plan = spec.plan
        self.spec = spec
        sk = plan.kernels[0]
        self.dtypes = [t.dtype for t in tensors]
        self.shapes = [t.shape for t in tensors]
        place = {op_id: n for n, op_id in enumerate(plan.inputs)}
        self.order = [place[o.op_id] for o in sk.operands]
        self.in_order = self.order == list(range(len(tensors)))
        self.out_shape, self.out_dtype = tuple(plan.output_shapes[0]), spec.out_dtypes[0]
        self.empty = torch.empty
        self.current_device = torch._C._cuda_getDevice
        self.current_stream = torch._C._cuda_getCurrentRawStream

    @staticmethod
    def fits(spec) -> bool:
        plan = spec.plan
        return (len(plan.kernels) == 1 and plan.kernels[0].family == "model" and not plan.temps
                and len(plan.outputs) == 1
                and len({o.op_id for o in plan.kernels[0].operands}) == len(plan.inputs)
                and all(d > 0 for d in plan.output_shapes[0]))

    def __call__(self, tensors):
        if len(tensors) != len(self.shapes):
            return NotImplemented
        device = tensors[0].get_device()
        if device < 0 or device != self.current_device():
            return NotImplemented
        for t, dtype, shape in zip(tensors, self.dtypes, self.shapes):
            if (t.dtype is not dtype or t.shape != shape or t.get_device() != device
                    or not t.is_contiguous() or t.data_ptr() % 16):
                return NotImplemented
        out = self.empty(self.out_shape, dtype=self.out_dtype, device=tensors[0].device)
        ins = tensors if self.in_order else [tensors[n] for n in self.order]
        _bound(self.spec, 0, device).run(ins, out, self.current_stream(device))
        return out


_native = None


def native_call():
    """The type ``Call`` of ``csrc/call.cpp``, or None where it is not built."""
    global _native
    if _native is None:
        from .build import call_library
        path = call_library()
        _native = False
        if path.exists():
            from importlib.machinery import ExtensionFileLoader
            from importlib.util import module_from_spec, spec_from_file_location
            loader = ExtensionFileLoader("molten_call", str(path))
            module = module_from_spec(spec_from_file_location("molten_call", str(path), loader=loader))
            loader.exec_module(module)
            _native = module.Call
    return _native or None


def short_call(spec, tensors, device: int):
    """The short way into ``spec``, whose plan is one model operator, for
    tensors like these (their shapes and types) on ``device``."""
    call = native_call()
    python = ModelCall(spec, tensors)
    b = _bound(spec, 0, device)
    short = b.short() if call else None
    if short is None:
        return python
    block, patches, maps = short
    lib, order = b.module.lib, python.order

    def address(fn):
        return ctypes.cast(fn, ctypes.c_void_p).value
    return call(address(lib.molten_launch), address(lib.molten_encode_tma_4d), b.module.handle.value, b.entry,
                bytes(b.cfg[1]), block,
                tuple((at, order[j] if j >= 0 else -1) for at, j in patches),
                tuple((at, order[j], *rest) for at, j, *rest in maps),
                tuple((t.dtype, tuple(t.shape)) for t in tensors), python.out_shape, python.out_dtype, device)
