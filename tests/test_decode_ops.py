"""The operators of a decode step without a GPU: shapes and refusals, launch
plans over their ranges, parameter blocks, and that their kernels compile."""
import ctypes
import random

import pytest

from molten_b200 import _capi, cli, decode, graphs
from molten_b200.build import build_cubin
from molten_b200.codegen import CodeGenerator, compile_graph
from molten_b200.fusion import FusionEngine
from molten_b200.ir import DataflowGraph, ModelOpType, OpType, TensorShape as TS
from molten_b200.lowering import LoweringError


def config_of(g, dtype, **tune):
    grp = FusionEngine().fuse(g)[0]
    k = CodeGenerator(dtype=dtype, tune=tune or None).generate(g, grp)
    assert [sk.family for sk in k.plan.kernels] == ["model"]
    return k.plan.kernels[0].config


def refused(g, text, dtype="bfloat16"):
    with pytest.raises(LoweringError, match=text):
        compile_graph(g, dtype=dtype)


# ------------------------------------------------------------------ refusals
def q4_graph(x, q, s, z=None, qdt="uint8", zdt="bfloat16"):
    g = DataflowGraph("q4")
    ids = [g.add_input("x", TS(x), dtype="bfloat16"), g.add_input("q", TS(q), dtype=qdt),
           g.add_input("s", TS(s), dtype="bfloat16")]
    zid = g.add_input("z", TS(z), dtype=zdt) if z else None
    g.add_output(g.matvec_q4(*ids, zeros=zid, name="y"))
    return g


@pytest.mark.parametrize("x,q,s,z,text", [
    ([1, 256], [64, 100], [64, 2], None, "nibbles"),
    ([1, 256], [64, 128], [63, 2], None, "scales"),
    ([1, 256], [64, 128], [64, 1], None, "scales"),            # groups of 256
    ([1, 96], [64, 48], [64, 1], None, "scales"),              # groups of 96
    ([1, 256], [64, 128], [64, 2], [64, 4], "zeros"),
    ([33, 256], [64, 128], [64, 2], None, "at most 32 rows"),
    ([3, 11, 256], [64, 128], [64, 2], None, "at most 32 rows"),
    ([1, 256], [64, 128, 1], [64, 2], None, "needs x"),
])
def test_matvec_q4_refusals(x, q, s, z, text):
    refused(q4_graph(x, q, s, z), text)


def test_matvec_q4_refuses_types():
    refused(q4_graph([1, 256], [64, 128], [64, 2], [64, 2], zdt="float32"), "one dtype")
    g = DataflowGraph("q4")
    x, q = g.add_input("x", TS([1, 256]), dtype="int32"), g.add_input("q", TS([64, 128]), dtype="uint8")
    s = g.add_input("s", TS([64, 2]), dtype="int32")
    g.add_output(g.matvec_q4(x, q, s))
    refused(g, "float type")


def rope_graph(x, tables, pos, sections=None, packed=False, style="half", x_dtype="bfloat16"):
    g = DataflowGraph("rope")
    xi = g.add_input("x", TS(x), dtype=x_dtype)
    c = g.add_input("cos", TS(tables), dtype="float32")
    s = None if packed else g.add_input("sin", TS(tables), dtype="float32")
    p = g.add_input("positions", TS(pos), dtype="int32")
    g.add_output(g.rope(xi, c, sin=s, style=style, positions=p, sections=sections))
    return g


@pytest.mark.parametrize("x,tables,pos,sections,text", [
    ([2, 8, 4, 63], [16, 31], [1, 2, 8], None, "even head_dim"),
    ([2, 8, 4, 64], [16, 64], [1, 2, 8], None, "rope table"),
    ([2, 8, 4, 64], [16, 32], [2, 2, 8], None, "positions of shape"),
    ([2, 8, 4, 64], [16, 32], [3, 2, 7], [16, 8, 8], "positions of shape"),
    ([2, 8, 4, 64], [16, 32], [2, 8], [16, 16], "positions of shape"),
    ([2, 8, 4, 64], [16, 32], [3, 2, 8], [16, 8, 4], "sections"),
    ([2, 8, 4, 64], [16, 32], [5, 2, 8], [16, 4, 4, 4, 4], "sections"),
    ([2, 8, 4, 64], [16, 32], [2, 2, 8], [36, -4], "sections"),
    ([4, 64], [16, 32], [1, 4], None, "rank >= 3"),
    ([2, 8, 4, 2048], [16, 1024], [1, 2, 8], None, "head_dim"),
])
def test_rope_positions_refusals(x, tables, pos, sections, text):
    refused(rope_graph(x, tables, pos, sections), text)


def test_rope_sections_need_positions_and_a_known_style():
    g = DataflowGraph("rope")
    x, f = g.add_input("x", TS([2, 8, 4, 64])), g.add_input("f", TS([8, 64]))
    with pytest.raises(ValueError, match="sections need positions"):
        g.rope(x, f, sections=[16, 16])
    refused(rope_graph([2, 8, 4, 64], [16, 32], [1, 2, 8], style="thirds"), "style")


def window_graph(q, k, v=None, lengths=None, dtype="bfloat16", v_dtype=None, **kw):
    g = DataflowGraph("window")
    ids = [g.add_input("q", TS(q), dtype=dtype), g.add_input("k", TS(k), dtype=dtype),
           g.add_input("v", TS(v or k), dtype=v_dtype or dtype)]
    n = g.add_input("lengths", TS(lengths), dtype="int32") if lengths else None
    g.add_output(g.window_attention(*ids, lengths=n, **kw))
    return g


@pytest.mark.parametrize("q,k,v,lengths,kw,text", [
    ([2, 1, 8, 64], [2, 10, 3, 64], None, None, {}, "8 heads over 3"),
    ([2, 1, 8, 64], [3, 10, 4, 64], None, None, {}, "needs q"),
    ([2, 1, 8, 64], [2, 10, 4, 32], None, None, {}, "needs q"),
    ([2, 1, 8, 64], [2, 10, 4, 64], [2, 11, 4, 64], None, {}, "needs q"),
    ([2, 1, 8, 60], [2, 10, 4, 60], None, None, {}, "multiple of 8"),
    ([2, 1, 8, 136], [2, 10, 4, 136], None, None, {}, "at most 128"),
    ([2, 1, 8, 64], [2, 0, 4, 64], None, None, {}, "at least one key"),
    ([2, 1, 8, 64], [2, 10, 4, 64], None, [3], {}, "lengths"),
    ([2, 1, 8, 64], [2, 10, 4, 64], None, None, {"window": 0}, "window 0"),
    ([2, 1, 8, 64], [2, 10, 4, 64], None, None, {"sinks": -1}, "sinks"),
    ([2, 1, 8, 64], [2, 10, 4, 64], None, None, {"scale": 0.0}, "positive"),
    ([2, 1, 8, 64], [2, 10, 4, 64], None, None, {"scale": float("inf")}, "positive"),
    ([2, 1, 8, 64], [2, 10, 4, 64], None, None, {"scale": float("nan")}, "positive"),
    ([1, 40, 256, 64], [1, 40, 1, 64], None, None, {}, "at most 128"),       # heads over one key head
])
def test_window_attention_refusals(q, k, v, lengths, kw, text):
    refused(window_graph(q, k, v, lengths, **kw), text)


def test_window_attention_takes_16_bit_types_only():
    refused(window_graph([1, 1, 2, 64], [1, 9, 2, 64], dtype="float32"), "bf16 or fp16", "float32")


def test_sample_refusals():
    def graph(logits, u, **params):
        g = DataflowGraph("sample")
        x, r = g.add_input("x", TS(logits), dtype="float32"), g.add_input("u", TS(u), dtype="float32")
        ids = {n: g.add_input(n, TS(s), dtype="float32" if n != "top_k" else "int32")
               for n, s in params.items()}
        g.add_output(g.sample(x, r, **ids))
        return g
    refused(graph([4, 100], [3]), "u of shape", "float32")
    refused(graph([100], []), "vocabulary", "float32")
    refused(graph([4, 100], [4], top_p=[5]), "top_p of shape", "float32")
    refused(graph([4, 100], [4], top_k=[4, 1]), "top_k of shape", "float32")
    refused(graphs.sample(1, 2 ** 20), "does not fit", "float32")
    compile_graph(graph([2, 2, 100], [2, 2], top_k=[2, 2]), dtype="float32")


def test_model_operators_do_not_take_scalar_operands():
    g = DataflowGraph("q4")
    x, q = g.add_input("x", TS([1, 256])), g.add_input("q", TS([64, 128]), dtype="uint8")
    c = g.add_constant("s", 1.0)
    g.add_output(g.add_op(ModelOpType.MATVEC_Q4, [x, q, c]))
    with pytest.raises(LoweringError):
        compile_graph(g, dtype="bfloat16")


# --------------------------------------------------------------------- plans
def test_q4_plans_over_the_range():
    rng = random.Random(1)
    for _ in range(150):
        group = rng.choice((32, 64, 128))
        k = group * rng.randint(1, 16384 // group)
        n, m = rng.choice((1, 15, 16, 17, rng.randint(1, 200000))), rng.randint(1, 32)
        dt = rng.choice(("bfloat16", "float16", "float32"))
        c = config_of(graphs.matvec_q4(m, n, k, group, dtype=dt, zeros=rng.random() < 0.5), dt)
        groups = k // group
        assert c["tiles"] * 16 * c["warps_n"] >= n > (c["tiles"] - 1) * 16 * c["warps_n"]
        assert c["warps"] % c["warps_n"] == 0 and c["ksplit"] <= groups
        assert 1 <= c["teams"] <= c["tiles"] or c["teams"] == 1
        assert c["tiles_per_cta"] * c["teams"] >= c["tiles"]
        assert c["chunk"] * c["ksplit"] >= groups or c["chunk"] >= 1
        assert c["smem"] <= decode.SMEM_LIMIT and (c["smem"] + 1024) * c["min_ctas"] <= decode.SMEM_SM + 4096


def test_q4_largest_rows_still_fit():
    for dt in ("bfloat16", "float32"):
        c = config_of(graphs.matvec_q4(32, 4096, 128 * 1000, 128, dtype=dt), dt)
        assert c["chunk"] < 1000 and c["smem"] <= decode.SMEM_LIMIT


def test_rope_plans_over_the_range():
    rng = random.Random(2)
    for _ in range(150):
        dim, heads = 2 * rng.randint(1, 512), rng.randint(1, 200)
        dt, style = rng.choice(("bfloat16", "float16", "float32")), rng.choice(("half", "interleaved"))
        c = config_of(graphs.rope_positions(rng.randint(1, 9), rng.randint(1, 5000), heads, dim, table=100,
                                            dtype=dt, style=style), dt)
        assert 1 <= c["block"] <= 1024
        assert c["block"] == c["head_lanes"] * c["tokens_per_cta"] * (
            dim // 2 // (c["vec"] if style == "half" else c["vec"] // 2))


def test_window_plans_over_the_range():
    rng = random.Random(3)
    for _ in range(200):
        per, kv = rng.choice((1, 2, 4, 5, 8, 32)), rng.randint(1, 16)
        new, cache = rng.choice((1, 2, 7, 33, 500, 8192)), rng.randint(1, 200000)
        dim = 8 * rng.randint(1, 16)
        c = config_of(graphs.window_attention(rng.randint(1, 64), new, cache, per * kv, kv, dim,
                                              window=rng.choice((None, 1, 100, 4096)),
                                              sinks=rng.choice((0, 1, 4, 200))), "bfloat16")
        assert (c["kind"] == "tiles") == (new * per > decode.WINDOW_FEW_ROWS)
        if c["kind"] == "tiles":
            assert 0 < c["positions"] * per <= 128 and c["blocks"] * 2 * c["positions"] >= new
            assert c["smem"] <= decode.SMEM_LIMIT
        else:
            assert 8 * c["nb"] >= c["rows"] and c["ranks"] in (1, 2, 4, 8)
            assert c["smem_launch"] <= decode.SMEM_LIMIT
            assert c["parts"] == 1 or c["ranks"] == 8


def test_window_wider_than_the_cache_is_none():
    for w in (4097, 10 ** 9):
        assert config_of(graphs.window_attention(1, 1, 4096, 8, 8, 64, window=w), "bfloat16")["window"] == -1
    assert config_of(graphs.window_attention(1, 1, 4096, 8, 8, 64, sinks=5000), "bfloat16")["sinks"] == 4096


def test_sample_plans_over_the_range():
    rng = random.Random(4)
    for _ in range(200):
        vocab, rows = int(2 ** rng.uniform(0, 18.3)), rng.randint(1, 2000)
        dt = rng.choice(("float32", "bfloat16", "float16"))
        c = config_of(graphs.sample(rows, vocab, dtype=dt), dt)
        word = 1 if dt == "float32" else 2
        assert c["block"] * c["run"] * c["ranks"] >= vocab
        assert c["run"] % word == 0 and c["run"] // word % 2 == 1
        assert c["block"] * c["run"] <= 65536 and c["smem"] <= decode.SMEM_LIMIT


def test_empty_batches_have_plans():
    for g, dt in ((graphs.matvec_q4(0, 64, 256, 64), "bfloat16"), (graphs.rope_positions(0, 4, 2, 64), "bfloat16"),
                  (graphs.rope_positions(2, 0, 2, 64), "bfloat16"), (graphs.window_attention(0, 1, 9, 4, 2, 64), "bfloat16"),
                  (graphs.window_attention(0, 90, 90, 4, 2, 64), "bfloat16"), (graphs.sample(0, 100), "float32")):
        assert config_of(g, dt)["block"] > 0


def test_sources_depend_on_types_not_sizes():
    def source(g, dt):
        return compile_graph(g, dtype=dt)[0].source
    # few rows: the warps of a CTA and its ring are in the source as well
    some = {source(graphs.window_attention(b, 1, cache, 32, 8, 128, window=w), "bfloat16")
            for b in (1, 3, 16, 64, 200) for cache in (100, 4096, 50000) for w in (None, 100, 3000)}
    assert len(some) <= 3
    assert (source(graphs.window_attention(1, 500, 4096, 32, 8, 128), "bfloat16")
            == source(graphs.window_attention(7, 64, 999, 16, 4, 72, window=None), "bfloat16"))
    a = compile_graph(graphs.sample(256, 100003), dtype="float32")[0]
    b = compile_graph(graphs.sample(300, 90000), dtype="float32")[0]
    assert a.source == b.source and a.plan.key != b.plan.key


# ----------------------------------------------------------- parameter blocks
def test_struct_layouts():
    assert ctypes.sizeof(_capi.Q4Args) == 88 and _capi.Q4Args.n.offset == 48
    assert ctypes.sizeof(_capi.RopePosArgs) == 120 and _capi.RopePosArgs.heads.offset == 80
    assert ctypes.sizeof(_capi.WindowArgs) == 168 and _capi.WindowArgs.batch.offset == 120
    assert ctypes.sizeof(_capi.WindowTcArgs) == 512 and _capi.WindowTcArgs.batch.offset == 440
    assert ctypes.sizeof(_capi.SampleArgs) == 96 and _capi.SampleArgs.rows.offset == 64


def test_tensor_map_arguments_are_checked():
    lib = _capi.load_library()
    buf = ctypes.create_string_buffer(256)
    at = (ctypes.addressof(buf) + 63) & ~63
    good = dict(tmap=at, dtype=_capi.DT_BF16, base=4096, dims=(128, 8, 100, 2), strides=(256, 2048, 204800),
                box=(64, 1, 128, 1))

    def call(**kw):
        a = dict(good, **kw)
        return lib.molten_encode_tma_4d(
            a["tmap"], a["dtype"], a["base"],
            a["dims"] and bytes((ctypes.c_uint64 * 4)(*a["dims"])),
            a["strides"] and bytes((ctypes.c_uint64 * 3)(*a["strides"])),
            a["box"] and bytes((ctypes.c_uint32 * 4)(*a["box"])))
    for bad in (dict(tmap=None), dict(base=None), dict(dims=None), dict(strides=None), dict(box=None),
                dict(tmap=at + 8), dict(base=4104), dict(dtype=7), dict(dims=(128, 0, 100, 2)),
                dict(dims=(128, 8, 2 ** 33, 2)), dict(strides=(256, 2040, 204800)),
                dict(strides=(0, 2048, 204800)), dict(strides=(256, 2048, 2 ** 40)),
                dict(box=(72, 1, 128, 1)), dict(box=(60, 1, 128, 1)), dict(box=(64, 1, 257, 1)),
                dict(box=(64, 0, 128, 1))):
        assert call(**bad) == 1, bad


# ------------------------------------------------------- kernels, JSON, reports
@pytest.mark.parametrize("graph,dtype", [
    (graphs.matvec_q4(1, 512, 512, 64), "bfloat16"),
    (graphs.matvec_q4(20, 512, 512, 32, dtype="float32", zeros=True), "float32"),
    (graphs.rope_positions(2, 8, 4, 128, sections=[16, 24, 24]), "bfloat16"),
    (graphs.window_attention(1, 1, 4096, 32, 8, 128), "bfloat16"),
    (graphs.window_attention(1, 100, 4096, 32, 8, 64, dtype="float16"), "float16"),
    (graphs.sample(2, 1000, top_k=True, top_p=0.9), "float32"),
])
def test_kernels_compile(graph, dtype, tmp_path):
    k = compile_graph(graph, dtype=dtype)[0]
    assert build_cubin(k.source, k.name, cache_dir=tmp_path).stat().st_size > 1000


def decode_graph():
    g = DataflowGraph("step")
    x = g.add_input("x", TS([2, 512]), dtype="bfloat16")
    w = g.add_input("w", TS([512]), dtype="bfloat16")
    q = g.add_input("q", TS([1000, 256]), dtype="uint8")
    s = g.add_input("s", TS([1000, 8]), dtype="bfloat16")
    u = g.add_input("u", TS([2]), dtype="float32")
    logits = g.matvec_q4(g.rms_norm(x, w, "norm"), q, s, name="logits")
    g.add_output(g.sample(logits, u, top_k=g.add_constant("k", 40), name="token"))
    return g


def test_json_round_trip_and_commands(tmp_path, capsys):
    import json
    for g in (graphs.sample(2, 100, top_k=50, top_p=True), decode_graph(),
              graphs.window_attention(1, 1, 64, 4, 2, 64), graphs.rope_positions(1, 4, 2, 64, sections=[8, 8, 16])):
        data = cli.graph_to_json(g)
        back = cli.graph_from_json(json.loads(json.dumps(data)))
        assert cli.graph_to_json(back) == data
        assert [o.op_type for o in back.ops.values()] == [o.op_type for o in g.ops.values()]
    p = tmp_path / "g.json"
    p.write_text(json.dumps(cli.graph_to_json(decode_graph())))
    assert cli.main(["compile", str(p), "-o", str(tmp_path / "out"), "--dtype", "bfloat16"]) == 0
    assert "kernel(s)" in capsys.readouterr().out
    text = "".join(f.read_text() for f in (tmp_path / "out").glob("molten_fused_*.cu"))
    assert "q4_matvec.cuh" in text and "sample.cuh" in text


def test_a_chain_keeps_its_order_and_types():
    ks = compile_graph(decode_graph(), dtype="bfloat16")
    fams = [sk.family for k in ks for sk in k.plan.kernels]
    assert fams.count("model") == 2 and fams[-1] == "model"
    out = ks[-1].plan.kernels[-1].outputs[0]
    assert out.dtype == "int32" and out.shape == (2,)


def test_a_token_cannot_enter_float_arithmetic():
    g = decode_graph()
    tok = g._outputs[-1]
    src = g.ops[tok].inputs[0] if g.ops[tok].op_type == OpType.OUTPUT else tok
    g.add_output(g.add_op(OpType.EXP, [src]))
    with pytest.raises(LoweringError):
        for k in compile_graph(g, dtype="bfloat16"):
            pass


# ------------------------------------------------------- the short host path
def test_short_call_checks_its_plan_and_its_tensors():
    torch = pytest.importorskip("torch")
    from molten_b200.build import build_call
    from molten_b200.decode_launch import native_call
    build_call()
    call, cfg = native_call(), bytes(_capi.LaunchCfg())
    assert call is not None
    x = ((torch.float32, (2, 3)),)
    good = [1, 1, 1, b"k", cfg, bytes(64), ((0, 0), (8, -1)), (), x, (2, 3), torch.float32, 0]
    c = call(*good)
    for where, bad in ((4, b"short"), (5, bytes(2000)), (6, ((60, 0),)), (6, ((0, 1),)), (6, ((-8, 0),)), (2, 0),
                       (7, ((0, 0, 1, bytes(32), bytes(24), bytes(16)),)), (7, ((0, 0, 1, b"", b"", b""),)),
                       (8, ((1, (2, 3)),)), (9, [2, 3]), (10, 5)):
        args = list(good)
        args[where] = bad
        with pytest.raises((ValueError, TypeError)):
            call(*args)
    # anything that is not a CUDA tensor of that type and shape: the general path
    for tensors in ((), (torch.zeros(2, 3),), (torch.zeros(3, 2),), (1,), (None,), (torch.nn.Parameter(torch.zeros(2, 3)),)):
        assert c(tensors) is NotImplemented
    with pytest.raises(TypeError):
        c(torch.zeros(2, 3))
    with pytest.raises(TypeError):
        c((), ())


# ------------------------------------------- which compiled kernel a graph gets
@pytest.fixture
def unbuilt(monkeypatch, tmp_path):
    """A runtime that builds no cubins."""
    from molten_b200 import runtime
    monkeypatch.setattr(runtime, "build_cubin", lambda source, name, *a, **kw: tmp_path / f"{name}.cubin")
    return runtime.MoltenRuntime(cache_dir=str(tmp_path))


def wired(order, build, shapes, dtypes):
    """A graph whose inputs are declared in ``order``."""
    g = DataflowGraph("wired")
    ids = {n: g.add_input(n, TS(shapes[n]), dtype=dtypes.get(n, "bfloat16")) for n in order}
    g.add_output(build(g, ids))
    return g


WIRED = {
    "window_attention": (("q", "k", "v"), ("q", "v", "k"), lambda g, i: g.window_attention(i["q"], i["k"], i["v"]),
                         {n: [1, 4, 2, 64] for n in "qkv"}, {}),
    "matvec_q4": (("x", "w", "s", "z"), ("x", "w", "z", "s"),
                  lambda g, i: g.matvec_q4(i["x"], i["w"], i["s"], zeros=i["z"]),
                  {"x": [2, 256], "w": [32, 128], "s": [32, 2], "z": [32, 2]}, {"w": "uint8"}),
    "rope_positions": (("x", "c", "s", "p"), ("x", "s", "c", "p"),
                       lambda g, i: g.rope(i["x"], i["c"], sin=i["s"], positions=i["p"]),
                       {"x": [2, 5, 2, 64], "c": [9, 32], "s": [9, 32], "p": [1, 2, 5]},
                       {"c": "float32", "s": "float32", "p": "int32"}),
    "sample": (("x", "u", "t", "p"), ("x", "u", "p", "t"),
               lambda g, i: g.sample(i["x"], i["u"], temperature=i["t"], top_p=i["p"]),
               {"x": [3, 100], "u": [3], "t": [3], "p": [3]}, {n: "float32" for n in "utp"}),
    "matmul": (("a", "b"), ("b", "a"), lambda g, i: g.matmul(i["a"], i["b"]), {n: [256, 256] for n in "ab"}, {}),
    "rope": (("x", "c", "s"), ("x", "s", "c"), lambda g, i: g.rope(i["x"], i["c"], sin=i["s"]),
             {"x": [1, 5, 2, 64], "c": [5, 32], "s": [5, 32]}, {}),
}


@pytest.mark.parametrize("name", WIRED)
def test_inputs_in_another_order_are_another_kernel(name, unbuilt):
    """The same source with its operands fed from other inputs."""
    first, second, build, shapes, dtypes = WIRED[name]
    ks = [compile_graph(wired(order, build, shapes, dtypes), dtype="bfloat16")[0] for order in (first, second, first)]
    cks = [unbuilt.compile(k) for k in ks]
    assert ks[0].source == ks[1].source
    assert cks[0] is not cks[1] and cks[0] is cks[2]
    for ck, k in zip(cks, ks):
        for a, b in zip(ck.kernel.plan.kernels, k.plan.kernels):
            assert [(o.index, o.op_id) for o in a.operands] == [(o.index, o.op_id) for o in b.operands]


@pytest.mark.parametrize("one,other", [
    (dict(window=None), dict(window=1000)), (dict(sinks=256), dict(sinks=5000)),
    (dict(scale=None), dict(scale=64 ** -0.5)), (dict(window=513), dict(window=None))])
def test_attributes_that_a_shape_hides_are_another_kernel(one, other, unbuilt):
    """A window wider than the declared cache is no limit there, but one in a
    longer cache: kernels are planned again for other shapes."""
    import torch
    from molten_b200 import runtime
    args = (2, 1, 256, 8, 2, 64)
    ks = [compile_graph(graphs.window_attention(*args, **kw), dtype="bfloat16")[0] for kw in (one, other, one)]
    assert ks[0].source == ks[1].source and ks[0].plan.kernels[0].config == ks[1].plan.kernels[0].config
    cks = [unbuilt.compile(k) for k in ks]
    assert cks[0] is not cks[1] and cks[0] is cks[2]
    # and each plans a longer cache, and wider heads, with its own attributes
    for ck, kw in zip(cks, (one, other)):
        tensors = [torch.empty(s, device="meta", dtype=t) for s, t in (
            ((2, 1, 8, 128), torch.bfloat16), ((2, 9000, 2, 128), torch.bfloat16), ((2, 9000, 2, 128), torch.bfloat16),
            ((2,), torch.int32))]
        got = ck.specialization(*tensors).plan.kernels[0].config
        want = config_of(graphs.window_attention(2, 1, 9000, 8, 2, 128, **kw), "bfloat16")
        assert got == want


# ------------------------------------------------------------------- clusters
@pytest.mark.parametrize("header,entry,first", [
    ("sample.cuh", "void sample_row(", "sm_combine<"), ("window_decode.cuh", "void window_decode(", "mapa.shared::cluster"),
    ("q4_matvec.cuh", "void q4_matvec(", "mapa.shared::cluster")])
def test_clusters_have_started_before_their_memory_is_used(header, entry, first):
    """Shared memory of another CTA of a cluster exists once that CTA runs: a
    kernel meets at a cluster barrier before its first access there."""
    from molten_b200.build import CSRC_DIR
    text = (CSRC_DIR / "include" / "molten" / header).read_text()
    body = text[text.index(entry):]
    before = body[:body.index(first)]
    assert "barrier.cluster.wait" in before or "q4_cluster_sync()" in before
    if "barrier.cluster.wait" in before:
        assert before.index("barrier.cluster.arrive") < before.index("barrier.cluster.wait")


# ------------------------------------------------ outputs in the inputs' memory
def check_overlap(g, dtype, tensors, outs):
    """What the runtime asks before a call writes to given outputs."""
    from molten_b200.decode_launch import refuse_overlap
    (k,) = compile_graph(g, dtype=dtype)
    names = [g.ops[i].name for i in k.plan.inputs]
    refuse_overlap(k.plan, [tensors[n] for n in names], outs)


@pytest.mark.parametrize("order", ["xcsp", "pcsx", "csxp", "cxsp"])
def test_rope_in_place_whatever_the_inputs_order(order):
    import torch
    shapes = {"x": [2, 5, 2, 64], "c": [40, 32], "s": [40, 32], "p": [1, 2, 5]}
    dtypes = {"x": "float32", "c": "float32", "s": "float32", "p": "int32"}
    g = wired(order, lambda g, i: g.rope(i["x"], i["c"], sin=i["s"], positions=i["p"]), shapes, dtypes)
    t = {n: torch.zeros(s, dtype=getattr(torch, dtypes[n])) for n, s in shapes.items()}
    check_overlap(g, "float32", t, [t["x"]])
    check_overlap(g, "float32", t, [torch.zeros_like(t["x"])])
    # over a table, from its start and from inside it
    for n in "cs":
        for at in (0, 8):
            t[n] = torch.zeros(2000)[at:at + 1280].view(40, 32)
            over = t[n].flatten().as_strided([2, 5, 2, 64], [640, 128, 64, 1])
            with pytest.raises(RuntimeError, match="overlaps"):
                check_overlap(g, "float32", t, [over])
    wide = torch.zeros(1288)
    t["x"] = wide[:1280].view(2, 5, 2, 64)
    with pytest.raises(RuntimeError, match="overlaps"):
        check_overlap(g, "float32", t, [wide[8:].view(2, 5, 2, 64)])


def test_overlaps_in_plans_of_several_kernels():
    import torch
    g = DataflowGraph("two")
    ids = {n: g.add_input(n, TS([1, 4, 2, 64]), dtype="bfloat16") for n in "rqkv"}
    q = g.add(ids["q"], ids["r"])
    g.add_output(q)
    g.add_output(g.window_attention(q, ids["k"], ids["v"]))
    t = {n: torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16) for n in "rqkv"}
    new = [torch.zeros_like(t["q"]) for _ in range(2)]
    check_overlap(g, "bfloat16", t, new)
    for n in "rq":                                     # (read before the attention writes, by nothing after)
        check_overlap(g, "bfloat16", t, [new[0], t[n]])
        check_overlap(g, "bfloat16", t, [t[n], new[1]])          # elementwise in place, as ever
    for n in "kv":
        for outs in ([new[0], t[n]], [t[n], new[1]], [new[0], t[n].flatten()[128:].as_strided([1, 4, 2, 64], [0, 96, 0, 1])]):
            with pytest.raises(RuntimeError, match="overlap"):
                check_overlap(g, "bfloat16", t, outs)
    with pytest.raises(RuntimeError, match="overlap"):
        check_overlap(g, "bfloat16", t, [new[0], new[0]])

    # x turned in place is read again by a later kernel
    g = DataflowGraph("turned")
    x = g.add_input("x", TS([1, 3, 2, 64]), dtype="float32")
    c = g.add_input("c", TS([9, 64]), dtype="float32")
    p = g.add_input("p", TS([1, 1, 3]), dtype="int32")
    y = g.rope(x, c, positions=p)
    g.add_output(y)
    g.add_output(g.add(y, x))
    t = {"x": torch.zeros(1, 3, 2, 64), "c": torch.zeros(9, 64), "p": torch.zeros(1, 1, 3, dtype=torch.int32)}
    with pytest.raises(RuntimeError, match="overlap"):
        check_overlap(g, "float32", t, [t["x"], torch.zeros_like(t["x"])])
    check_overlap(g, "float32", t, [torch.zeros_like(t["x"]), t["x"]])


def test_overlap_is_left_to_plans_without_model_operators():
    import torch
    g = DataflowGraph("plain")
    x = g.add_input("x", TS([4, 64]), dtype="float32")
    g.add_output(g.silu(x))
    t = torch.zeros(4, 64)
    check_overlap(g, "float32", {"x": t}, [t])


def test_rope_reads_x_as_memory_that_it_may_write():
    """.nc loads are for memory that nothing writes while the kernel runs, and
    RoPE at positions may turn x in place."""
    import re
    from molten_b200.build import CSRC_DIR
    inc = CSRC_DIR / "include" / "molten"
    body = (inc / "rope_positions.cuh").read_text()
    body = body[body.index("void rope_positions("):]
    assert set(re.findall(r"load_slot<(\w+), XT", body)) == {"kLoadInPlace"}
    common = (inc / "common.cuh").read_text()
    for part in common.split("== kLoadInPlace")[1:]:
        assert ".nc" not in part[:part.index("} else")] and "__ldg" not in part[:part.index("} else")]


# ----------------------------------------------------------- what shapes share
def test_shapes_and_runtimes_share_modules(monkeypatch, tmp_path):
    """A source that holds for all sizes is loaded once on a device."""
    import torch
    from molten_b200 import runtime
    loads = []

    class Module:
        def __init__(self, path, device):
            loads.append((path, device))
    monkeypatch.setattr(runtime, "build_cubin", lambda source, name, *a, **kw: tmp_path / f"{name}.cubin")
    monkeypatch.setattr(runtime._capi, "Module", Module)
    monkeypatch.setattr(runtime, "_loaded", {})
    k = compile_graph(graphs.sample(1, 32768, top_k=True), dtype="float32")[0]
    for rt in (runtime.MoltenRuntime(cache_dir=str(tmp_path)), runtime.MoltenRuntime(cache_dir=str(tmp_path))):
        ck = rt.compile(k)
        for rows in range(1, 11):
            spec = ck._spec_for([torch.empty(s, device="meta", dtype=t) for s, t in (
                ((rows, 32768), torch.float32), ((rows,), torch.float32), ((rows,), torch.float32),
                ((rows,), torch.int32))])
            assert spec.gk.source == k.source
            assert spec.module(0) is spec.module(0) is not spec.module(1)
    assert sorted(loads) == [(str(tmp_path / f"{k.name}.cubin"), d) for d in (0, 1)]


def test_the_number_of_kept_shapes_is_bounded(monkeypatch, unbuilt):
    import torch
    from molten_b200 import runtime
    monkeypatch.setattr(runtime, "MAX_SHAPES", 8)
    ck = unbuilt.compile(compile_graph(graphs.matvec_q4(1, 64, 256, 64), dtype="bfloat16")[0])

    def spec_of(m):
        return ck._spec_for([torch.empty(s, device="meta", dtype=t) for s, t in (
            ((m, 256), torch.bfloat16), ((64, 128), torch.uint8), ((64, 4), torch.bfloat16))])
    for turn in range(2):
        for m in range(1, 20):
            spec = spec_of(m)
            assert spec is spec_of(m) and spec.plan.output_shapes == [(m, 64)]
            assert len(ck._specs) <= 8


def test_headers_are_read_again_where_they_changed(monkeypatch, tmp_path):
    from molten_b200 import build
    (tmp_path / "molten").mkdir()
    a, b = tmp_path / "molten" / "a.cuh", tmp_path / "molten" / "b.cuh"
    a.write_text("one")
    b.write_text("two")
    monkeypatch.setattr(build, "ENGINE_INCLUDE", tmp_path)
    seen = [build._engine_digest()]
    assert build._engine_digest() == seen[0]
    for change in (lambda: a.write_text("longer"), lambda: b.unlink(), lambda: b.write_text("2"), lambda: b.rename(a)):
        change()
        seen.append(build._engine_digest())
    assert len(set(seen)) == len(seen)


def test_one_source_is_looked_up_once(monkeypatch, tmp_path):
    import torch
    from molten_b200 import runtime
    built = []
    monkeypatch.setattr(runtime, "build_cubin", lambda source, name, *a, **kw: built.append(source) or tmp_path / "x.cubin")
    rt = runtime.MoltenRuntime(cache_dir=str(tmp_path))
    ck = rt.compile(compile_graph(graphs.sample(1, 32768), dtype="float32")[0])
    for rows in range(0, 9):
        ck._spec_for([torch.empty(s, device="meta") for s in ((rows, 32768), (rows,), (rows,))])
    assert len(built) == 1
    rt.clear_cache()
    rt.compile(ck.kernel)
    assert len(built) == 2


@pytest.mark.parametrize("failure", [FileNotFoundError("g++"), "BuildError"])
def test_kernels_are_built_without_the_short_host_path(failure, monkeypatch, capsys, tmp_path):
    """The native short path has a complete fallback: what it needs besides nvcc
    does not keep the kernels from being built."""
    import __graft_entry__ as entry
    from molten_b200 import build
    from oracle import build_ref
    built = []

    def fails(*a, **kw):
        raise build.BuildError("torch/extension.h") if failure == "BuildError" else failure
    monkeypatch.setattr(build, "build_call", fails)
    monkeypatch.setattr(build, "build_runtime", lambda *a, **kw: built.append("runtime"))
    monkeypatch.setattr(build, "build_cubin", lambda source, name, *a, **kw: built.append(name))
    monkeypatch.setattr(build_ref, "build", lambda *a, **kw: None)
    entry.build()
    assert "runtime" in built and len(built) > 10
    assert "short host path was not built" in capsys.readouterr().err


# --------------------------------------------- parameters by name and by number
@pytest.mark.parametrize("params", [[], ["temperature"], ["topk", "top_p"], ["top_k", "top_k"], ["top_k", "top_p", "min_p"],
                                    "top_k", None])
def test_sample_parameters_that_do_not_fit_its_inputs(params):
    """Inputs without a name, or with one that is not known, would be left out."""
    g = DataflowGraph("sample")
    x, u = g.add_input("x", TS([4, 100]), dtype="float32"), g.add_input("u", TS([4]), dtype="float32")
    k, p = g.add_input("k", TS([4]), dtype="int32"), g.add_input("p", TS([4]), dtype="float32")
    attrs = {} if params is None else {"params": params}
    g.add_output(g.add_op(ModelOpType.SAMPLE, [x, u, k, p], "token", **attrs))
    refused(g, "sample: parameters", "float32")


@pytest.mark.parametrize("value,text", [(float("nan"), "top_k"), (float("inf"), "top_k"), (2.5, "top_k")])
def test_sample_top_k_is_a_whole_number(value, text):
    refused(graphs.sample(4, 100, top_k=value), text, "float32")


def test_sample_top_k_past_32_bits_is_no_limit():
    from molten_b200.decode_launch import _Sample
    for value, want in ((40, 40), (40.0, 40), (2 ** 31 - 1, 2 ** 31 - 1), (2 ** 32 + 5, 2 ** 31 - 1), (-2 ** 40, -1), (0, 0)):
        (k,) = compile_graph(graphs.sample(4, 100, top_k=value), dtype="float32")
        bound = object.__new__(_Sample)
        bound.c, a = k.plan.kernels[0].config, _capi.SampleArgs()
        bound.fill(a)
        assert min(a.top_k_all, 100) == min(want, 100) and (a.top_k_all > 0) == (want > 0)


def test_json_attributes_beside_the_type():
    """Attributes of these operators may stand beside the type, as eps may."""
    ops = [{"type": "INPUT", "name": n, "inputs": [], "shape": s, "dtype": "bfloat16"}
           for n, s in (("q", [1, 1, 4, 64]), ("k", [1, 90, 2, 64]), ("v", [1, 90, 2, 64]))]
    ops += [{"type": "WINDOW_ATTENTION", "inputs": [0, 1, 2], "window": 20, "sinks": 3, "scale": 0.5},
            {"type": "OUTPUT", "inputs": [3]}]
    g = cli.graph_from_json({"name": "a", "ops": ops})
    assert config_of(g, "bfloat16") == config_of(
        graphs.window_attention(1, 1, 90, 4, 2, 64, window=20, sinks=3, scale=0.5, lengths=False), "bfloat16")
    ops = [{"type": "INPUT", "name": n, "inputs": [], "shape": s, "dtype": d}
           for n, s, d in (("x", [1, 5, 2, 64], "bfloat16"), ("f", [9, 64], "float32"), ("p", [2, 1, 5], "int32"))]
    ops += [{"type": "ROTATE_POSITIONS", "inputs": [0, 1, 2], "sections": [20, 12], "style": "half", "packed": True},
            {"type": "OUTPUT", "inputs": [3]}]
    c = config_of(cli.graph_from_json({"name": "a", "ops": ops}), "bfloat16")
    assert c["sections"] == [20, 12] and c["half"] and c["packed"]


@pytest.mark.parametrize("name", ["temperature", "top_k", "top_p", "min_p"])
def test_sample_parameters_are_vectors_or_constants(name):
    """A tensor of no dimension holds one number, not one a row."""
    g = DataflowGraph("sample")
    x, u = g.add_input("x", TS([4, 100]), dtype="float32"), g.add_input("u", TS([4]), dtype="float32")
    p = g.add_input(name, TS([]), dtype="int32" if name == "top_k" else "float32")
    g.add_output(g.sample(x, u, **{name: p}))
    refused(g, f"{name} of shape", "float32")


def test_sample_parameters_of_a_call_are_vectors(unbuilt):
    import torch
    ck = unbuilt.compile(compile_graph(graphs.sample(4, 100), dtype="float32")[0])
    good = [torch.empty(s, device="meta") for s in ((4, 100), (4,), (4,))]
    ck._spec_for(good)
    for shape in ((), (1,), (5,), (4, 1)):
        with pytest.raises(LoweringError):
            ck._spec_for(good[:2] + [torch.empty(shape, device="meta")])


@pytest.mark.parametrize("kind", ["window_attention", "rms_norm"])
def test_equal_layers_share_a_kernel(kind, unbuilt):
    """Groups that differ in their op numbers alone, as the layers of a model."""
    def kernel(before):
        g = DataflowGraph("layer")
        for n in range(before):                        # (used by nothing: later numbers)
            g.add_input(f"other{n}", TS([4, 64]), dtype="bfloat16")
        if kind == "window_attention":
            ids = [g.add_input(n, TS([1, 4, 2, 64]), dtype="bfloat16") for n in "qkv"]
            y = g.window_attention(*ids, window=3)
        else:
            y = g.rms_norm(g.add_input("x", TS([4, 512]), dtype="bfloat16"),
                           g.add_input("w", TS([512]), dtype="bfloat16"), "norm")
        g.add_output(y)
        (k,) = compile_graph(g, dtype="bfloat16")
        return k
    a, b = kernel(0), kernel(3)
    assert a.source == b.source and a.plan.inputs != b.plan.inputs
    assert unbuilt.compile(a) is unbuilt.compile(b)
