"""Parameter blocks and launches of the model operators (``decode.py``).

Every call reads pointers, strides and sizes from the tensors it is given;
nothing is kept from one call for the next.  Workspaces come from torch's
allocator on the launching stream, one per call, so calls on several streams
and captured graphs never share one.
"""

from __future__ import annotations

import ctypes
import math

from . import _capi
from .decode import SMS
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


def _aligned(t, nbytes: int, strides) -> bool:
    return t.data_ptr() % nbytes == 0 and all(s * t.element_size() % nbytes == 0 for s in strides)


def _check_aligned(name: str, entry: bytes, t, nbytes: int) -> None:
    if t.data_ptr() % nbytes:
        raise _capi.MoltenError(f"input {name!r} at {t.data_ptr():#x} is not {nbytes}-byte aligned "
                                f"as kernel {entry.decode()} requires")


def _cfg(grid, block: int, cluster: int = 1, smem: int = 0):
    from .runtime import PDL
    cfg = _capi.LaunchCfg()
    cfg.grid[:] = [grid, 1, 1]
    cfg.block[:] = [block, 1, 1]
    cfg.cluster[:] = [cluster, 1, 1]
    cfg.smem_bytes = smem
    cfg.flags = _capi.LAUNCH_PDL if PDL else 0
    return cfg


def launch_model_op(spec, i: int, env: dict, device: int, stream: int) -> None:
    """Launch sub-kernel ``i`` of ``spec`` on ``stream``."""
    sk = spec.plan.kernels[i]
    ins = {o.index: env[o.op_id] for o in sk.operands}
    _LAUNCH[sk.config["op"]](spec, sk, spec.entries[i], ins, env[sk.outputs[0].op_id], device, stream)


def _launch_q4(spec, sk, entry, ins, out, device, stream):
    c = sk.config
    x, q, scales, zeros = _merged(ins[0], 1), ins[1], ins[2], ins.get(3)
    if not _aligned(x, 16, x.stride()[:-1]) and x.shape[0] > 1:
        x = x.contiguous()
    _check_aligned(sk.operands[0].name, entry, x, 16)
    _check_aligned(sk.operands[1].name, entry, q, 16)
    for o, t in zip(sk.operands[2:], (scales, zeros)):
        _check_aligned(o.name, entry, t, DTYPE_SIZE[o.dtype])
    a = _capi.Q4Args()
    a.x, a.q, a.scales, a.out = x.data_ptr(), q.data_ptr(), scales.data_ptr(), out.data_ptr()
    a.zeros = zeros.data_ptr() if zeros is not None else None
    a.x_stride, a.n, a.m, a.k = x.stride(0), c["n"], c["m"], c["k"]
    a.warps_n_log, a.ksplit_log = c["warps_n"].bit_length() - 1, c["ksplit"].bit_length() - 1
    a.chunk, a.tiles, a.teams = c["chunk"], c["tiles"], c["teams"]
    cfg = _cfg(c["teams"] * c["ksplit"], c["block"], c["ksplit"], c["smem"])
    spec.module(device).launch(entry, cfg, a, stream)


def _launch_rope(spec, sk, entry, ins, out, device, stream):
    c = sk.config
    x = _merged(ins[0], 2)
    tables, pos = [ins[j] for j in range(1, len(ins) - 1)], ins[len(ins) - 1]
    if c["xvec"]:
        slot = min(16, c["vec"] * x.element_size())
        if not _aligned(x, slot, x.stride()[:-1]):
            x = x.contiguous()
        _check_aligned(sk.operands[0].name, entry, x, slot)
        _check_aligned("output", entry, out, min(16, c["vec"] * out.element_size()))
    if c["tvec"]:
        for o, t in zip(sk.operands[1:], tables):
            _check_aligned(o.name, entry, t, c["table_slot"])
    a = _capi.RopePosArgs()
    a.x, a.cos_t, a.pos, a.out = x.data_ptr(), tables[0].data_ptr(), pos.data_ptr(), out.data_ptr()
    a.sin_t = tables[-1].data_ptr()
    a.status = _capi.status_word(device)
    a.tokens, a.x_token, a.x_head = c["tokens"], x.stride(0), x.stride(1)
    a.table_rows, a.heads, a.dim = c["table_rows"], c["heads"], c["dim"]
    a.axes, a.head_lanes, a.tokens_per_cta = len(c["sections"]), c["head_lanes"], c["tokens_per_cta"]
    end = 0
    for j, width in enumerate(c["sections"]):
        end += width
        a.bound[j] = end
    grid = -(-c["tokens"] // c["tokens_per_cta"])
    spec.module(device).launch(entry, _cfg(grid, c["block"]), a, stream)


def _tma_4d(t, dtype: str, box) -> bytes:
    """TMA descriptor of t [b, s, h, d]; the stride of a dim of one element
    (any number in torch) is replaced by one that the encoder takes."""
    b, s, h, d = t.shape
    size = t.element_size()
    strides = [t.stride(2) if h > 1 else 8, t.stride(1) if s > 1 else 8, t.stride(0) if b > 1 else 8]
    return _capi.encode_tma_4d(_capi.DT_BF16 if dtype == "bfloat16" else _capi.DT_F16, t.data_ptr(),
                               (d, h, s, b), [x * size for x in strides], box)


def _launch_window_tiles(spec, sk, entry, q, k, v, lengths, out, device, stream):
    c = sk.config
    dt = sk.operands[0].dtype
    a = _capi.WindowTcArgs()
    ctypes.memmove(a.tmap_q, _tma_4d(q, dt, (64, c["per"], c["positions"], 1)), 128)
    ctypes.memmove(a.tmap_k, _tma_4d(k, dt, (64, 1, 128, 1)), 128)
    ctypes.memmove(a.tmap_v, _tma_4d(v, dt, (64, 1, 128, 1)), 128)
    a.v, a.out = v.data_ptr(), out.data_ptr()
    a.lengths = lengths.data_ptr() if lengths is not None else None
    a.status = _capi.status_word(device)
    a.v_b, a.v_s, a.v_h = v.stride()[:3]
    a.batch, a.nq, a.cache, a.kv_heads = c["batch"], c["new"], c["cache"], c["kv_heads"]
    a.per, a.dim, a.window, a.sinks = c["per"], c["dim"], c["window"], c["sinks"]
    a.scale_log2, a.positions, a.blocks = c["scale"] * LOG2E, c["positions"], c["blocks"]
    spec.module(device).launch(entry, _cfg(min(c["items"], SMS), c["block"], 1, c["smem"]), a, stream)


def _launch_window(spec, sk, entry, ins, out, device, stream):
    c = sk.config
    a = _capi.WindowArgs()
    qkv = []
    for j in range(3):
        t = ins[j]
        # 16-byte rows: the last dim contiguous, every other stride a multiple
        # of 8 elements (and not 0 where the tiles are copied by TMA)
        if ((t.stride(3) != 1 and t.shape[3] > 1) or not _aligned(t, 16, t.stride()[:3])
                or (c["kind"] == "tiles" and any(n > 1 and x == 0 for n, x in zip(t.shape, t.stride())))):
            t = t.contiguous()
        _check_aligned(sk.operands[j].name, entry, t, 16)
        qkv.append(t)
    q, k, v = qkv
    _check_aligned("output", entry, out, 16)
    if c["kind"] == "tiles":
        _launch_window_tiles(spec, sk, entry, q, k, v, ins.get(3), out, device, stream)
        return
    a.q, a.k, a.v, a.out = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
    a.lengths = ins[3].data_ptr() if 3 in ins else None
    a.q_b, a.q_s, a.q_h = q.stride()[:3]
    a.k_b, a.k_s, a.k_h = k.stride()[:3]
    a.v_b, a.v_s, a.v_h = v.stride()[:3]
    a.batch, a.nq, a.cache, a.kv_heads = c["batch"], c["new"], c["cache"], c["kv_heads"]
    a.per, a.dim, a.window, a.sinks = c["per"], c["dim"], c["window"], c["sinks"]
    a.scale_log2 = c["scale"] * LOG2E
    a.ranks, a.parts = c["ranks"], c["parts"]
    mod = spec.module(device)
    grid = c["items"] * c["parts"] * c["ranks"]
    part = None
    if c["parts"] > 1:
        import torch
        part = torch.empty(c["items"] * c["parts"] * c["rows"] * (c["dim"] + 2),
                           dtype=torch.float32, device=q.device)
        a.part = part.data_ptr()
    mod.launch(entry, _cfg(grid, c["block"], c["ranks"], c["smem_launch"]), a, stream)
    if part is not None:
        mod.launch(entry + b"_join", _cfg(-(-c["items"] * c["rows"] // 4), 128), a, stream)


def _launch_sample(spec, sk, entry, ins, out, device, stream):
    c = sk.config
    x = _merged(ins[0], 1)
    _check_aligned(sk.operands[0].name, entry, x, x.element_size())
    a = _capi.SampleArgs()
    a.logits, a.u, a.out = x.data_ptr(), ins[1].data_ptr(), out.data_ptr()
    a.row_stride, a.rows, a.vocab = x.stride(0), c["rows"], c["vocab"]
    a.run, a.ranks = c["run"], c["ranks"]
    a.temperature_all, a.top_p_all = 1.0, 1.0        # without a parameter: no limit
    for i, name in enumerate(c["params"]):
        if 2 + i in ins:
            setattr(a, name, ins[2 + i].data_ptr())
        else:
            value = c["scalars"][2 + i]
            setattr(a, name + "_all", int(value) if name == "top_k" else float(value))
    spec.module(device).launch(entry, _cfg(c["rows"] * c["ranks"], c["block"], c["ranks"], c["smem"]), a,
                               stream)


_LAUNCH = {ModelOpType.MATVEC_Q4: _launch_q4, ModelOpType.ROTATE_POSITIONS: _launch_rope,
           ModelOpType.WINDOW_ATTENTION: _launch_window, ModelOpType.SAMPLE: _launch_sample}

# operands a kernel takes as strided views; the rest are made contiguous
STRIDED = {ModelOpType.MATVEC_Q4: (0,), ModelOpType.ROTATE_POSITIONS: (0,),
           ModelOpType.WINDOW_ATTENTION: (0, 1, 2), ModelOpType.SAMPLE: (0,)}
