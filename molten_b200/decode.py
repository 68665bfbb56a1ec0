"""The operators of a decode step: shapes, launch plans and CUDA emission.

``ModelOpType`` (``ir.py``) adds to the graph what answering a batch of
requests needs next to RMSNorm, RoPE and the GEMM:

* ``MATVEC_Q4``         products of a few rows with 4-bit weights;
* ``ROTATE_POSITIONS``  RoPE at given positions, on up to four axes;
* ``WINDOW_ATTENTION``  attention over a sliding window and the first keys;
* ``SAMPLE``            temperature, top-k, top-p and min-p from given numbers.

Each runs as a sub-kernel of family ``model`` (``lowering.split_group``).
Unlike the row, elementwise and GEMM families, their sources are
instantiations of the engine headers with types and head sizes only: batch
sizes, lengths and strides travel in the parameter block, so every shape runs
from the same few cubins and inputs may be strided views.
``decode_launch.py`` fills the parameter blocks.
"""

from __future__ import annotations

from .ir import DataflowGraph, ModelOpType, OpType
from .lowering import (
    DTYPE_CTYPE, DTYPE_SIZE, INT_DTYPES, LoweringError, Operand, OutputSpec, ROPE_STYLES,
    SubKernel, prod,
)

SMS = 148                         # streaming multiprocessors of a B200

Q4_GROUPS = (32, 64, 128)
Q4_MAX_ROWS = 32
Q4_MAX_KSPLIT = 8                 # portable cluster size
Q4_SUMS_BYTES = 16 * 1024         # sums of a CTA's tiles, where they are kept
SMEM_LIMIT = 227 * 1024           # shared memory of a CTA, and of an SM
SMEM_SM = 228 * 1024

WINDOW_MAX_DIM = 128
WINDOW_FEW_ROWS = 32              # rows of a key head up to which the few-row kernel runs
WINDOW_STAGES, WINDOW_TILE = 3, 16

SAMPLE_FIXED = 2 * 8 * 24 + 32 * 24 + 2048 + 4096 + 2 * 2048 + 64   # of SampleShared (molten/sample.cuh)

SAMPLE_PARAMS = ("temperature", "top_k", "top_p", "min_p")

ROPE_MAX_AXES = 4
ROPE_MAX_DIM = 1024


def _need(ok, text: str) -> None:
    if not ok:
        raise LoweringError(text)


# ------------------------------------------------------------------- shapes
def infer_shape(op, ins: list) -> tuple:
    """Result shape of a model operator; raises on shapes it does not take."""
    ins = [tuple(int(d) for d in s) for s in ins]
    return _SHAPES[op.op_type](op, ins)


def _q4_shape(op, ins):
    _need(len(ins) in (3, 4), "matvec_q4 takes (x, qweight, scales[, zeros])")
    x, q, s = ins[:3]
    _need(len(x) >= 1 and len(q) == 2 and len(s) == 2,
          f"matvec_q4 needs x [..., K], qweight [N, K/2], scales [N, K/G]: {x}, {q}, {s}")
    k, n = x[-1], q[0]
    _need(k > 0 and q[1] * 2 == k, f"matvec_q4: qweight {q} does not pack K = {k} nibbles a row")
    _need(s[0] == n and s[1] > 0 and k % s[1] == 0 and k // s[1] in Q4_GROUPS,
          f"matvec_q4: scales {s} for [{n}, {k}] weights; groups of {Q4_GROUPS}")
    _need(len(ins) == 3 or ins[3] == s, f"matvec_q4: zeros {ins[-1]} and scales {s} differ in shape")
    return x[:-1] + (n,)


def _rope_shape(op, ins):
    packed = bool(op.attrs.get("packed"))
    _need(len(ins) == (3 if packed else 4), "rope with positions takes (x, tables, positions)")
    x, pos = ins[0], ins[-1]
    _need(len(x) >= 3, f"rope needs x of rank >= 3 ([..., seq, heads, head_dim]), got {x}")
    d, lead = x[-1], x[:-2]
    _need(d % 2 == 0 and 0 < d <= ROPE_MAX_DIM,
          f"rope needs an even head_dim of at most {ROPE_MAX_DIM}, got {d}")
    _need((op.attrs.get("style") or "interleaved") in ROPE_STYLES,
          f"rope style {op.attrs.get('style')!r} (interleaved, half)")
    width = d if packed else d // 2
    for t in ins[1:-1]:
        _need(len(t) == 2 and t[0] > 0 and t[1] == width and t == ins[1],
              f"rope table of shape {t}; expected [rows, {width}]")
    sections = op.attrs.get("sections") or [d // 2]
    _need(1 <= len(sections) <= ROPE_MAX_AXES and all(v >= 0 for v in sections)
          and sum(sections) == d // 2,
          f"rope sections {sections} must be at most {ROPE_MAX_AXES} counts of pairs with sum {d // 2}")
    want = (len(sections),) + lead
    _need(pos == want or (len(sections) == 1 and pos == lead),
          f"rope positions of shape {pos}; expected {want}")
    return x


def _window_shape(op, ins):
    _need(len(ins) in (3, 4), "window_attention takes (q, k, v[, lengths])")
    q, k, v = ins[:3]
    _need(len(q) == 4 and len(k) == 4 and k == v and q[0] == k[0] and q[3] == k[3],
          "window_attention needs q [batch, new, heads, d] and k, v [batch, cache, kv_heads, d]: "
          f"{q}, {k}, {v}")
    _need(k[1] > 0, "window_attention needs a cache of at least one key")
    _need(k[2] > 0 and q[2] % k[2] == 0, f"window_attention: {q[2]} heads over {k[2]} key heads")
    _need(0 < q[3] <= WINDOW_MAX_DIM and q[3] % 8 == 0,
          f"window_attention: head dim {q[3]} must be a multiple of 8, at most {WINDOW_MAX_DIM}")
    _need(len(ins) == 3 or ins[3] == q[:1], f"window_attention: lengths {ins[-1]}, expected {q[:1]}")
    scale = op.attrs.get("scale")
    _need(scale is None or 0 < scale < float("inf"), f"window_attention: scale {scale} must be positive")
    w, s = op.attrs.get("window"), op.attrs.get("sinks") or 0
    _need(w is None or w >= 1, f"window_attention: window {w} must be at least 1 (None: no limit)")
    _need(s >= 0, f"window_attention: {s} sinks")
    return q


def _sample_shape(op, ins):
    _need(len(ins) >= 2, "sample takes (logits, u[, parameters])")
    logits, u = ins[:2]
    _need(len(logits) >= 2 and logits[-1] > 0, f"sample needs logits [..., vocabulary], got {logits}")
    lead = logits[:-1]
    _need(u == lead, f"sample: u of shape {u}, expected {lead}")
    params = op.attrs.get("params") or ()
    _need(isinstance(params, (list, tuple)) and len(params) == len(ins) - 2 and len(set(params)) == len(params)
          and set(params) <= set(SAMPLE_PARAMS),
          f"sample: parameters {params!r} for {len(ins) - 2} inputs behind logits and u; each one of {SAMPLE_PARAMS}")
    for name, s in zip(params, ins[2:]):
        _need(s in ((), lead), f"sample: {name} of shape {s}, expected {lead} or a constant")
    return lead


_SHAPES = {ModelOpType.MATVEC_Q4: _q4_shape, ModelOpType.ROTATE_POSITIONS: _rope_shape,
           ModelOpType.WINDOW_ATTENTION: _window_shape, ModelOpType.SAMPLE: _sample_shape}


# -------------------------------------------------------------------- types
def _slot_dtypes(op) -> dict:
    """Operand position -> the dtype it has to have."""
    t = op.op_type
    if t == ModelOpType.MATVEC_Q4:
        return {1: "uint8"}
    if t == ModelOpType.ROTATE_POSITIONS:
        return {len(op.inputs) - 1: "int32"}
    if t == ModelOpType.WINDOW_ATTENTION:
        return {3: "int32"} if len(op.inputs) > 3 else {}
    slots = {1: "float32"}
    for i, p in enumerate(op.attrs.get("params", ())):
        slots[2 + i] = "int32" if p == "top_k" else "float32"
    return slots


def fixed_input_dtypes(graph: DataflowGraph) -> dict:
    """Graph inputs whose dtype an operator fixes (positions, lengths, packed
    weights, random numbers ...), and the tables and scales, which keep the
    dtype they are declared with."""
    out = {}
    for op in graph.ops.values():
        if not isinstance(op.op_type, ModelOpType):
            continue
        slots = dict(_slot_dtypes(op))
        if op.op_type == ModelOpType.MATVEC_Q4:
            declared = range(2, len(op.inputs))
        elif op.op_type == ModelOpType.ROTATE_POSITIONS:
            declared = range(1, len(op.inputs) - 1)
        else:
            declared = ()
        for i, src in enumerate(op.inputs):
            if graph.ops[src].op_type != OpType.INPUT:
                continue
            if i in slots:
                out[src] = slots[i]
            elif i in declared:
                out[src] = graph.ops[src].dtype
    return out


# ------------------------------------------------------------------ planning
def plan_model_op(graph, op_id: int, outs, shapes: dict, dts: dict, tune: dict) -> SubKernel:
    """SubKernel of one model operator for concrete shapes and dtypes.  Its
    ``config`` holds ``op`` (the operator), ``block``, ``flops`` and what the
    launch needs; scalar operands are in ``config["scalars"]``."""
    op = graph.ops[op_id]
    _need(list(outs) == [op_id], f"the {op.op_type.name} sub-kernel has one output")
    slots = _slot_dtypes(op)
    operands, scalars = [], {}
    for pos, j in enumerate(op.inputs):
        src = graph.ops[j]
        if src.op_type == OpType.CONSTANT:
            _need(op.op_type == ModelOpType.SAMPLE and pos >= 2
                  and isinstance(src.attrs.get("value"), (int, float)),
                  f"{op.op_type.name}: operand {pos} must be a tensor")
            scalars[pos] = src.attrs["value"]
            continue
        want = slots.get(pos)
        if want:
            _need(dts[j] == want, f"{op.op_type.name}: operand {src.name or pos!r} is {dts[j]}, "
                                  f"expected {want}")
        else:
            _need(dts[j] not in INT_DTYPES,
                  f"{op.op_type.name}: operand {src.name or pos!r} is {dts[j]}, expected a float type")
        operands.append(Operand(index=pos, op_id=j, name=src.name or f"op{j}", dtype=dts[j],
                                shape=tuple(shapes[j]), last="vec", row_map="full"))
    outputs = [OutputSpec(index=0, op_id=op_id, dtype=dts[op_id], shape=tuple(shapes[op_id]),
                          kind="full")]
    sk = SubKernel(family="model", op_ids=[op_id], operands=operands, outputs=outputs)
    sk.config = {"op": op.op_type, "scalars": scalars}
    sk.config.update(_PLANS[op.op_type](op, sk, tune or {}))
    return sk


def _plan_q4(op, sk, tune) -> dict:
    x, q, s = sk.operands[:3]
    k, n = x.shape[-1], q.shape[0]
    m = max(1, prod(x.shape[:-1]))                    # (no rows: planned as one, not launched)
    _need(m <= Q4_MAX_ROWS, f"matvec_q4 takes at most {Q4_MAX_ROWS} rows of x, got {m}")
    _need(k < 2 ** 31 and n < 2 ** 31 - 512, "matvec_q4: sizes beyond 2^31")
    if len(sk.operands) == 4:
        _need(sk.operands[3].dtype == s.dtype, "matvec_q4: zeros and scales must have one dtype")
    group = k // s.shape[1]
    nt = 1 if m <= 8 else (2 if m <= 16 else 4)
    o = tune.get("q4") or {}
    groups, w = s.shape[1], group // 32
    planes = 3 if x.dtype == "float32" else 1

    def layout(warps, warps_n, ksplit, occupancy):
        """One way to run it, or None: warps of a CTA, of these along the rows
        of q, CTAs of a cluster along k, CTAs of an SM."""
        # the warps of a CTA split k, as far as there are groups for them
        while "warps_n" not in o and warps_n < warps and warps // warps_n > groups:
            warps_n *= 2
        tiles = -(-n // (16 * warps_n))
        limit = (SMEM_SM // occupancy - 1024) // 1024 * 1024
        per_cta = -(-groups // ksplit)                # groups of one CTA
        if ksplit > groups:                           # (one would have none)
            return None
        group_bytes = m * (planes * 64 * w + 8)
        fixed = 16 + 2 * warps * nt * 128 * 4
        sums = warps_n * 16 * m * 4                   # of one tile
        # x is staged whole where it fits, else in the fewest equal chunks
        chunk, chunks = per_cta, 1
        if fixed + per_cta * group_bytes + (Q4_SUMS_BYTES if ksplit > 1 else 0) > limit:
            room = limit - Q4_SUMS_BYTES - fixed
            if room < group_bytes:
                return None
            chunks = -(-per_cta // (room // group_bytes))
            chunk = -(-per_cta // chunks)
        keep = chunks > 1 or ksplit > 1               # tiles' sums stay in shared memory
        teams = max(1, min(tiles, SMS * occupancy // ksplit))
        if keep:
            teams = max(teams, -(-tiles // max(1, Q4_SUMS_BYTES // sums)))
        tiles_per_cta = -(-tiles // teams)
        smem = fixed + chunk * group_bytes + (tiles_per_cta * sums if keep else 0)
        if smem > SMEM_LIMIT:
            return None
        # microseconds, from 850 measured layouts of 23 shapes (one in six off by a
        # third): the first term is instructions issued, the next two a warp's
        # latency a group, then staging x by the SM and by a CTA, a tile's end, and
        # what splitting k over CTAs costs
        waves = -(-teams * ksplit // (SMS * occupancy))
        ctas = min(occupancy, -(-teams * ksplit // SMS))
        rounds = tiles_per_cta * waves
        warps_k = warps // warps_n
        steps = rounds * sum(-(-min(chunk, per_cta - i * chunk) // warps_k) for i in range(chunks))
        columns, staged = nt * planes, waves * per_cta * m * group * planes
        split = ksplit.bit_length() - 1
        cost = (0.0103 * ctas * warps * steps * columns + (0.071 * w + 0.18) * steps
                + staged * (0.045 * ctas / 1024 + 1.66 / (2048 * warps)) + 1.09 * chunks * waves
                + rounds * (0.24 * chunks + 0.0083 * ctas * warps * columns + 0.01 * keep * m)
                + (1.14 + 0.42 * (rounds - 1)) * split + (0.17 * rounds if split else 0.0))
        return cost, {"m": m, "n": n, "k": k, "group": group, "nt": nt, "warps": warps, "warps_n": warps_n,
                      "tiles": tiles, "ksplit": ksplit, "depth": int(o.get("depth") or 2),
                      "zeros": len(sk.operands) == 4, "chunk": chunk, "min_ctas": occupancy, "teams": teams,
                      "tiles_per_cta": tiles_per_cta, "smem": smem, "block": 32 * warps,
                      "flops": 2 * m * n * k}

    # 24 warps an SM only with one column block of one plane (registers)
    shapes = [(8, 3), (8, 2), (16, 1)] if nt == 1 and planes == 1 else [(8, 2), (16, 1)]
    ways = [layout(int(o.get("warps") or warps), int(o.get("warps_n") or warps_n), int(o.get("ksplit") or ksplit),
                   int(o.get("occupancy") or occupancy))
            for warps, occupancy in shapes for warps_n in (1, 2, 4)
            for ksplit in (1, 2, 4, 8) if ksplit <= Q4_MAX_KSPLIT]
    ways = [way for way in ways if way]
    _need(ways, f"matvec_q4: {m} rows of K = {k} do not fit")
    return min(ways, key=lambda way: way[0])[1]


def _plan_rope(op, sk, tune) -> dict:
    packed = bool(op.attrs.get("packed"))
    style = op.attrs.get("style") or "interleaved"
    x, pos, out = sk.operands[0], sk.operands[-1], sk.outputs[0]
    tables = sk.operands[1:-1]
    _need(packed or tables[0].dtype == tables[1].dtype, "rope: cos and sin must have one dtype")
    d, heads = x.shape[-1], x.shape[-2]
    tokens = prod(x.shape[:-2])
    _need(tokens < 2 ** 31 and heads < 2 ** 31, "rope: sizes beyond 2^31")
    sections = op.attrs.get("sections") or [d // 2]
    half = style == "half"
    span = d // 2 if half else d
    o = tune.get("rope") or {}
    vec = 16 // min(DTYPE_SIZE[x.dtype], DTYPE_SIZE[out.dtype])
    while vec > 1 and span % vec:
        vec //= 2
    if not half:
        vec = max(vec, 2)
    xvec = o.get("vec") != 1 and not (vec == 1 or vec * DTYPE_SIZE[x.dtype] < 4)
    pairs = vec if half else vec // 2
    slot = pairs * (2 if packed else 1) * DTYPE_SIZE[tables[0].dtype]      # table bytes per slot
    row = tables[0].shape[1] * DTYPE_SIZE[tables[0].dtype]
    tvec = xvec and row % min(16, slot) == 0 and slot in (2, 4, 8, 16, 32, 64)
    spr = (d // 2) // pairs
    # heads per thread (measured, 1 / 2 / 4 / 8: bf16 half-style [2, 4700, 22,
    # 128] 21.0 / 16.9 / 23.0 / 29.4 us, [48, 1, 40, 128] 2.6 / 2.1 / 3.2, fp32
    # interleaved [2, 4096, 32, 128] 46.0 / 43.7 / 42.0 / 42.3)
    hpt = int(o.get("heads") or min(heads, 2))
    lanes = max(1, min(-(-heads // hpt), 256 // spr if spr <= 256 else 1))
    per_cta = max(1, 256 // (spr * lanes))
    return {"dim": d, "heads": heads, "tokens": tokens, "sections": list(sections), "vec": vec,
            "xvec": xvec, "tvec": tvec, "half": half, "packed": packed, "hpt": hpt,
            "head_lanes": lanes, "tokens_per_cta": per_cta, "block": spr * lanes * per_cta,
            "table_rows": tables[0].shape[0], "table_slot": min(16, slot),
            "flops": 3 * tokens * heads * d}


def _split_window(items: int, tiles: int, most_warps: int):
    """(ranks, parts, warps): how the keys of an item (``tiles`` tiles of 16)
    are spread over the CTAs of a cluster, over clusters, and over the warps
    of a CTA.  An SM holds 8 warps; a CTA costs about 4 us to fill and drain
    and 1.4 us per tile of each warp, a join of parts 2.5 us and more
    (measured with head dim 128, 4 rows: 8 items of 66 tiles 6.6 us on 8 CTAs
    of 8 warps each, 12-17 us on one or two; 512 items of 257 tiles 154 us on
    one CTA of 4 warps each, 170 of 2, 161 of 8; 8 items of 4096 tiles 54 us
    on 4 x 8 CTAs of 4 warps, 114 on 8; 1 item of 512 tiles 11.5 us on 4 x 8
    CTAs, 18 on 8).  CTAs of 8 warps in large numbers leave SMs without a
    place for a whole cluster."""
    best = None
    for warps in (4, 8, 2):
        slots = SMS * (8 // warps)
        for ranks in (1, 2, 4, 8):
            for parts in (1, 2, 4) if ranks == 8 else (1,):
                ctas = items * ranks * parts
                if warps > most_warps or warps == 8 and ranks > 1 and ctas > 64:
                    continue
                per_warp = -(-tiles // (ranks * parts * warps))
                waves = 1.0 if ctas <= slots else ctas / slots + 0.15
                cost = waves * (4.0 + 1.4 * per_warp) + (2.5 + 0.2 * parts if parts > 1 else 0.0)
                if best is None or cost < best[0] - 1e-9:
                    best = (cost, ranks, parts, warps)
    return best[1:]


def _plan_window(op, sk, tune) -> dict:
    q, k, v = sk.operands[:3]
    _need(q.dtype == k.dtype == v.dtype and q.dtype in ("bfloat16", "float16"),
          f"window_attention takes bf16 or fp16 q, k and v of one type, got {q.dtype}, {k.dtype}, "
          f"{v.dtype}")
    batch, new, heads, dim = q.shape
    cache, kv_heads = k.shape[1], k.shape[2]
    per = heads // kv_heads
    rows, items = new * per, batch * kv_heads
    _need(max(cache, new) < 2 ** 30 and items < 2 ** 24 and rows < 2 ** 30,
          "window_attention: sizes beyond the kernel's range")
    window, sinks = op.attrs.get("window"), op.attrs.get("sinks") or 0
    window = -1 if window is None or window >= cache + new else window
    sinks = min(sinks, cache)
    scale = op.attrs.get("scale")
    scale = dim ** -0.5 if scale is None else scale
    o = tune.get("window") or {}
    c = {"batch": batch, "new": new, "cache": cache, "kv_heads": kv_heads, "per": per, "dim": dim,
         "window": window, "sinks": sinks, "scale": scale, "dp": 64 if dim <= 64 else 128}
    # most keys a row can see, and most keys any row of a request sees
    seen = cache if window < 0 else min(cache, window + sinks)
    span = cache if window < 0 else min(cache, window + sinks + new)
    c["flops"] = 4 * batch * heads * new * seen * dim
    if o.get("kind") == "tiles" or (o.get("kind") is None and rows > WINDOW_FEW_ROWS):
        return _plan_window_tiles(c, o)
    tiles = -(-span // WINDOW_TILE) + 1
    nb = 1 if rows <= 8 else 2 if rows <= 16 else 4
    ranks, parts, warps = _split_window(items, tiles, 8 if nb == 1 else 4)
    ranks, parts = int(o.get("ranks") or ranks), int(o.get("parts") or parts)
    warps = int(o.get("warps") or warps)
    # what the ranks of a cluster send one another: 16 bytes per 2 columns
    inbox = -(-rows * (dim // 2) // ranks) * ranks * 16 if ranks > 1 else 0
    area = warps * 8 * nb * (c["dp"] + 4) * 4
    # 8 warps an SM, twice that where a tile is half as wide; a third stage
    # where the SM's shared memory holds it
    min_ctas = max(1, min(4, 8 // warps)) * (2 if c["dp"] == 64 and nb < 4 else 1)
    for stages in (WINDOW_STAGES, WINDOW_STAGES - 1):
        stages = int(o.get("stages") or stages)
        ring = warps * stages * 2 * WINDOW_TILE * c["dp"] * 2
        smem = max(ring, area) + warps * 8 * nb * (8 + WINDOW_TILE * 4)
        if (smem + inbox + 1024) * min_ctas <= SMEM_SM:
            break
    _need(smem + inbox <= SMEM_LIMIT, "window_attention: the tile does not fit shared memory")
    c.update(kind="few", nb=nb, ranks=ranks, parts=parts, items=items, rows=rows, warps=warps,
             stages=stages, min_ctas=min_ctas, block=32 * warps, smem=smem, smem_launch=smem + inbox)
    return c


def _plan_window_tiles(c: dict, o: dict) -> dict:
    """The tcgen05 kernel: pairs of Q tiles of up to 128 (position, head) rows."""
    per, dp = c["per"], c["dp"]
    _need(per <= 128, f"window_attention: {per} heads over one key head; at most 128")
    positions = 128 // per
    blocks = -(-c["new"] // (2 * positions))
    items = c["batch"] * c["kv_heads"] * blocks
    _need(items < 2 ** 31, "window_attention: sizes beyond the kernel's range")
    dch = dp // 64
    stages = int(o.get("stages") or (5 if dp == 128 else 10))
    bars = 3 * stages + 17
    smem = 2 * dch * 16384 + stages * dch * 16384 + bars * 8 + 48 + 1024
    _need(smem <= SMEM_LIMIT, f"window_attention: {stages} stages need {smem} bytes")
    # fewer items than SMs: CTAs share an item's key tiles, at least two each (a
    # tile takes some 1.9 us, the join some 5)
    span = c["cache"] if c["window"] < 0 else min(c["cache"], c["window"] + c["sinks"] + 2 * positions)
    tiles = span // 128 + 2
    parts = max(1, min(SMS // max(items, 1), tiles // 2, 32))
    parts = int(o.get("parts") or (parts if parts > 1 and tiles > 5 else 1))
    _need(parts <= 32, f"window_attention: {parts} parts; at most 32")
    _need(items * parts < 2 ** 31 // 256, "window_attention: sizes beyond the kernel's range")
    c.update(kind="tiles", positions=positions, blocks=blocks, items=items, stages=stages,
             smem=smem, block=384, ranks=1, parts=parts)
    return c


def _sample_fixed(dtype, threads) -> int:
    packed = threads * 32 // DTYPE_SIZE[dtype]        # tokens: value and 16-bit index
    return SAMPLE_FIXED + packed * (DTYPE_SIZE[dtype] + 2)


def _plan_sample(op, sk, tune) -> dict:
    logits = sk.operands[0]
    vocab, rows = logits.shape[-1], prod(logits.shape[:-1])
    _need(rows * 8 < 2 ** 31, "sample: sizes beyond 2^31")
    for o in sk.operands[2:]:                         # (constants have no shape: infer_shape takes them)
        _need(o.shape == logits.shape[:-1], f"sample: {op.attrs['params'][o.index - 2]} of shape {o.shape}, expected "
                                            f"{logits.shape[:-1]} or a constant")
    for pos, value in sk.config["scalars"].items():
        _need(op.attrs["params"][pos - 2] != "top_k" or value == value // 1,
              f"sample: top_k {value} is not a whole number")
    o = tune.get("sample") or {}

    word = 4 // DTYPE_SIZE[logits.dtype]              # tokens of 32 bits

    def run_of(threads, ranks):
        # consecutive tokens of a thread: an odd number of words (no bank conflicts)
        return word * (-(-vocab // (threads * ranks * word)) | 1)

    def smem_of(threads, ranks):
        return (_sample_fixed(logits.dtype, threads)
                + threads * run_of(threads, ranks) * DTYPE_SIZE[logits.dtype] + 16)

    def ranks_of(threads, at_once):
        # the fewest CTAs a row that leave room for 768 threads on an SM; more
        # where threads have many tokens and all rows still run at once (30 x
        # 50257: 4 CTAs of 512 threads a row 42.0 us, 8 52.4; 16 x 131072: 68.5 and
        # 50.9; 100 x 20000: 4 of 256 threads 46.9, 2 54.5)
        ranks = 1
        while ranks < 8 and (smem_of(threads, ranks) > SMEM_SM * threads // 768 - 1024
                             or (rows * ranks * 2 <= at_once and run_of(threads, ranks) > 24)):
            ranks *= 2
        return ranks
    # 512 threads where all rows run at once without long runs (128 x 8000: 23.5
    # us, 256 threads 32.9; 100 x 20000: 55 and 46.9); a few clusters more than SMs
    # still count as at once
    wide = ranks_of(512, SMS * 11 // 10)
    few = rows * wide <= SMS * 11 // 10 and (wide == 8 or run_of(512, wide) <= 36)
    threads = int(o.get("threads") or (512 if few else 256))
    ranks = int(o.get("ranks") or (wide if few and threads == 512 else ranks_of(threads, SMS * 28 // 10)))
    # (a token's index within its CTA's part has 16 bits)
    _need(smem_of(threads, ranks) <= SMEM_LIMIT and threads * run_of(threads, ranks) <= 65536,
          f"sample: a vocabulary of {vocab} does not fit the shared memory of a cluster")
    return {"rows": rows, "vocab": vocab, "ranks": ranks, "run": run_of(threads, ranks),
            "smem": smem_of(threads, ranks), "block": threads,
            "min_ctas": int(o.get("min_ctas") or max(1, 768 // threads)), "params": list(op.attrs.get("params", ())),
            "flops": 2 * rows * vocab}


_PLANS = {ModelOpType.MATVEC_Q4: _plan_q4, ModelOpType.ROTATE_POSITIONS: _plan_rope,
          ModelOpType.WINDOW_ATTENTION: _plan_window, ModelOpType.SAMPLE: _plan_sample}


def launch_record(sk: SubKernel) -> dict:
    c = sk.config
    rec = {"op": c["op"].name.lower(), "block": c["block"], "smem": c.get("smem", 0)}
    if c["op"] == ModelOpType.MATVEC_Q4:
        rec.update(grid=c["teams"] * c["ksplit"], cluster=c["ksplit"], warps_n=c["warps_n"])
    elif c["op"] == ModelOpType.ROTATE_POSITIONS:
        rec.update(head_lanes=c["head_lanes"], tokens_per_cta=c["tokens_per_cta"])
    elif c["op"] == ModelOpType.SAMPLE:
        rec.update(grid=c["rows"] * c["ranks"], cluster=c["ranks"])
    elif c["op"] == ModelOpType.WINDOW_ATTENTION:
        if c["kind"] == "tiles":
            rec.update(kind="tiles", positions=c["positions"], blocks=c["blocks"], items=c["items"],
                       parts=c["parts"])
        else:
            rec.update(kind="few", cluster=c["ranks"], parts=c["parts"], smem=c["smem_launch"],
                       grid=c["items"] * c["parts"] * c["ranks"])
    return rec


# ------------------------------------------------------------------ emission
def emit_model_op(sk: SubKernel, name: str) -> str:
    return _EMIT[sk.config["op"]](sk, name)


def _bool(v) -> str:
    return "true" if v else "false"


def _emit_q4(sk, name):
    c = sk.config
    xt, st = (DTYPE_CTYPE[sk.operands[i].dtype] for i in (0, 2))
    ot = DTYPE_CTYPE[sk.outputs[0].dtype]
    return f"""// Molten sm_100a 4-bit matrix-vector product: {name}
// x {sk.operands[0].dtype}, groups of {c['group']}, up to {8 * c['nt']} rows
#include "molten/q4_matvec.cuh"

using namespace molten;

extern "C" __global__ void __launch_bounds__({c['block']}, {c['min_ctas']}) {name}(const __grid_constant__ Q4Args args) {{
  extern __shared__ __align__(16) uint8_t smem_raw[];
  pdl_enter();
  q4_matvec<{xt}, {st}, {ot}, {c['group']}, {c['nt']}, {_bool(c['zeros'])}, {c['depth']}, {c['warps']}>(args, smem_raw);
}}
"""


def _emit_rope(sk, name):
    c = sk.config
    xt, tt = (DTYPE_CTYPE[sk.operands[i].dtype] for i in (0, 1))
    ot = DTYPE_CTYPE[sk.outputs[0].dtype]
    return f"""// Molten sm_100a RoPE at given positions: {name}
// x {sk.operands[0].dtype}, {'packed table' if c['packed'] else 'tables'} {sk.operands[1].dtype}
#include "molten/rope_positions.cuh"

using namespace molten;

extern "C" __global__ void __launch_bounds__(1024) {name}(const __grid_constant__ RopePosArgs args) {{
  pdl_enter();
  rope_positions<{xt}, {tt}, {ot}, {c['vec']}, {_bool(c['half'])}, {_bool(c['packed'])}, {_bool(c['xvec'])}, {_bool(c['tvec'])}, {c['hpt']}>(args);
}}
"""


def _emit_window(sk, name):
    c = sk.config
    t, ot = DTYPE_CTYPE[sk.operands[0].dtype], DTYPE_CTYPE[sk.outputs[0].dtype]
    if c["kind"] == "tiles":
        return f"""// Molten sm_100a window attention: {name}
// {sk.operands[0].dtype}, head dim up to {c['dp']}
#include "molten/window_sm100.cuh"

using namespace molten;

typedef WindowTcLayout<{c['dp']}, {c['stages']}> Layout_{name};
static_assert(Layout_{name}::SMEM_BYTES == {c['smem']}, "the launch's dynamic shared memory");
static_assert(Layout_{name}::THREADS == {c['block']}, "block size");

extern "C" __global__ void __launch_bounds__({c['block']}, 1) {name}(const __grid_constant__ WindowTcArgs args) {{
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const WindowTcShared sh = window_tc_carve<Layout_{name}>(smem_raw);
  window_tc_init<Layout_{name}>(sh, args);     // mbarriers + TMEM allocation
  pdl_enter();                                 // no global access before this
  __syncthreads();
  window_tc_roles<Layout_{name}, {t}, {ot}, {_bool(c['parts'] > 1)}>(sh, args);
  tc_fence_before();
  __syncthreads();
  window_tc_teardown<Layout_{name}>(sh);       // TMEM release
}}

extern "C" __global__ void __launch_bounds__(256) {name}_join(const __grid_constant__ WindowTcArgs args) {{
  pdl_enter();
  window_tc_join<{ot}>(args);
}}
"""
    lay = f"{c['dp']}, {c['nb']}, {c['warps']}, {c['stages']}"
    return f"""// Molten sm_100a window attention, few query rows: {name}
// {sk.operands[0].dtype}, head dim up to {c['dp']}, up to {8 * c['nb']} rows
#include "molten/window_decode.cuh"

using namespace molten;

static_assert(WindowDecodeLayout<{lay}>::SMEM == {c['smem']}, "the launch's dynamic shared memory");

extern "C" __global__ void __launch_bounds__({c['block']}, {c['min_ctas']}) {name}(const __grid_constant__ WindowArgs args) {{
  extern __shared__ __align__(128) uint8_t smem_raw[];
  pdl_enter();
  window_decode<{t}, {ot}, {lay}>(args, smem_raw);
}}

extern "C" __global__ void __launch_bounds__(128) {name}_join(const __grid_constant__ WindowArgs args) {{
  pdl_enter();
  window_join<{ot}>(args);
}}
"""


def _emit_sample(sk, name):
    t = DTYPE_CTYPE[sk.operands[0].dtype]
    return f"""// Molten sm_100a sampling: {name}
// {sk.operands[0].dtype} logits
#include "molten/sample.cuh"

using namespace molten;

static_assert(sizeof(SampleShared<{t}, {sk.config['block']}>) == {_sample_fixed(sk.operands[0].dtype, sk.config['block'])}, "the launch's dynamic shared memory");

extern "C" __global__ void __launch_bounds__({sk.config['block']}, {sk.config['min_ctas']}) {name}(const __grid_constant__ SampleArgs args) {{
  extern __shared__ __align__(16) uint8_t smem_raw[];
  sample_table<{t}, {sk.config['block']}>(smem_raw);
  pdl_enter();
  sample_row<{t}, {sk.config['block']}>(args, smem_raw);
}}
"""


_EMIT = {ModelOpType.MATVEC_Q4: _emit_q4, ModelOpType.ROTATE_POSITIONS: _emit_rope,
         ModelOpType.WINDOW_ATTENTION: _emit_window, ModelOpType.SAMPLE: _emit_sample}
