"""The operators of a decode step used together on a B200: a layer and its
sampling in eager calls and in captured graphs, several streams, repeated
tensors, empty batches, and tensors past 2^31 elements."""
import pytest

torch = pytest.importorskip("torch")

from molten_b200 import _capi, graphs
from molten_b200.codegen import compile_graph
from molten_b200.ir import DataflowGraph, OpType, TensorShape as TS
from molten_b200.runtime import MoltenRuntime

from .test_decode_ops_gpu import (
    DEV, DT, attention_inputs, check_attention, check_q4, check_rope, check_sample, compiled, gen_of,
    half_step, q4_inputs, q4_reference, sample_inputs, tables, window_kernel)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rt():
    return MoltenRuntime()


# -------------------------------------------------------------- a decode step
BATCH, HIDDEN, HEADS, KV, DIM, CACHE, VOCAB, GROUP = 3, 512, 8, 2, 64, 200, 5003, 64
WINDOW, SINKS = 50, 2


class Step:
    """One layer and the sampling of one new token per request."""

    def __init__(self, rt):
        def q4(n, seed):
            return q4_inputs(1, n, HIDDEN, GROUP, "bfloat16", True, seed)[1:]
        self.qkv, self.out, self.head = q4((HEADS + 2 * KV) * DIM, 1), q4(HIDDEN, 2), q4(VOCAB, 3)
        g = gen_of(4)
        self.norms = [(1 + 0.1 * torch.randn(HIDDEN, generator=g, device=DEV)).bfloat16() for _ in range(2)]
        self.cos, self.sin = tables(CACHE, DIM // 2)
        self.k = torch.randn(BATCH, CACHE, KV, DIM, generator=g, device=DEV).bfloat16()
        self.v = torch.randn(BATCH, CACHE, KV, DIM, generator=g, device=DEV).bfloat16()

        def product(name, n, norm, sample=False, residual=False):
            g = DataflowGraph(name)
            x = g.add_input("x", TS([BATCH, HIDDEN]), dtype="bfloat16")
            y = x
            if norm:
                w = g.add_input("w", TS([HIDDEN]), dtype="bfloat16")
                y = g.rms_norm(x, w, "norm")
            q = g.add_input("q", TS([n, HIDDEN // 2]), dtype="uint8")
            s = g.add_input("s", TS([n, HIDDEN // GROUP]), dtype="bfloat16")
            z = g.add_input("z", TS([n, HIDDEN // GROUP]), dtype="bfloat16")
            y = g.matvec_q4(y, q, s, zeros=z, name="product")
            if residual:
                y = g.add(y, g.add_input("r", TS([BATCH, HIDDEN]), dtype="bfloat16"))
            if sample:
                g.add_output(y)
                u = g.add_input("u", TS([BATCH]), dtype="float32")
                y = g.sample(y, u, temperature=g.add_constant("t", 0.8), top_k=g.add_constant("k", 50),
                             top_p=g.add_constant("p", 0.9))
            g.add_output(y)
            ks = [rt.compile(k) for k in compile_graph(g, dtype="bfloat16")]
            return g, ks
        self.first = product("first", (HEADS + 2 * KV) * DIM, True)
        self.last = product("last", HIDDEN, False, residual=True)
        self.pick = product("pick", VOCAB, True, sample=True)
        self.rope_q = compiled(rt, graphs.rope_positions(BATCH, 1, HEADS, DIM, table=CACHE), "bfloat16")
        self.rope_k = compiled(rt, graphs.rope_positions(BATCH, 1, KV, DIM, table=CACHE), "bfloat16")
        self.attend = window_kernel(rt, BATCH, 1, CACHE, HEADS, KV, DIM, WINDOW, SINKS, "bfloat16")

    @staticmethod
    def chain(graph_kernels, *tensors):
        """Run a graph's kernels in order (each takes inputs and earlier outputs)."""
        g, ks = graph_kernels
        env = dict(zip((i for i in sorted(g.ops) if g.ops[i].op_type == OpType.INPUT), tensors))
        for k in ks:
            plan = k.kernel.plan
            res = k(*[env[i] for i in plan.inputs])
            env.update(zip(plan.outputs, res if isinstance(res, tuple) else (res,)))
        return [env[o if o in env else g.ops[o].inputs[0]] for o in g._outputs]

    def __call__(self, x, positions, lengths, slots, u):
        seen = {}
        (qkv,) = self.chain(self.first, x, self.norms[0], *self.qkv)
        q, k, v = qkv.view(BATCH, 1, -1, DIM).split([HEADS, KV, KV], 2)       # strided views
        seen["qkv"], seen["q"], seen["k"] = qkv, q, k
        qr, kr = self.rope_q(q, self.cos, self.sin, positions), self.rope_k(k, self.cos, self.sin, positions)
        at = torch.arange(BATCH, device=DEV)
        self.k[at, slots] = kr[:, 0]
        self.v[at, slots] = v[:, 0]
        a = self.attend(qr, self.k, self.v, lengths)
        (y,) = self.chain(self.last, a.view(BATCH, HIDDEN), *self.out, x)
        logits, token = self.chain(self.pick, y, self.norms[1], *self.head, u)
        seen.update(qr=qr, kr=kr, a=a, y=y, logits=logits, token=token)
        return seen


def step_inputs(n):
    g = gen_of(50 + n)
    x = torch.randn(BATCH, HIDDEN, generator=g, device=DEV).bfloat16()
    lengths = torch.tensor([1 + n, 60 + n, CACHE - 3 + n], dtype=torch.int32, device=DEV)
    slots = (lengths - 1).long()
    return [x, (lengths - 1).view(1, BATCH, 1).contiguous(), lengths, slots,
            torch.rand(BATCH, generator=g, device=DEV)]


def norm_of(x, w):
    xd = x.double()
    return xd * torch.rsqrt((xd * xd).mean(-1, keepdim=True) + 1e-6) * w.double()


def test_decode_step(rt):
    step = Step(rt)
    for n in range(3):
        x, pos, lengths, slots, u = step_inputs(n)
        s = step(x, pos, lengths, slots, u)
        # RMSNorm and product: the normalised row is rounded once to bf16 in
        # between, half a step of each term
        want = norm_of(x, step.norms[0])
        ref, mag = q4_reference(want, *step.qkv)
        tol = half_step("bfloat16") * ref.abs() + (1.01 * half_step("bfloat16") + 2.0 ** -18) * mag
        assert bool(((s["qkv"].double() - ref).abs() <= tol).all())
        check_rope(s["qr"], s["q"], step.cos, step.sin, pos, [DIM // 2], "half", "bfloat16")
        check_rope(s["kr"], s["k"], step.cos, step.sin, pos, [DIM // 2], "half", "bfloat16")
        check_attention(s["a"], s["qr"], step.k, step.v, lengths, WINDOW, SINKS, "bfloat16", 2.0 ** -16)
        ref, mag = q4_reference(s["a"].view(BATCH, HIDDEN), *step.out)
        ref = ref + x.double()
        # the product is rounded before the sum, and the sum again
        tol = half_step("bfloat16") * (ref.abs() + 1.01 * (ref - x.double()).abs()) + 2.0 ** -18 * mag
        assert bool(((s["y"].double() - ref).abs() <= 1.01 * tol).all())
        ref, mag = q4_reference(norm_of(s["y"], step.norms[1]), *step.head)
        tol = half_step("bfloat16") * ref.abs() + (1.01 * half_step("bfloat16") + 2.0 ** -18) * mag
        assert bool(((s["logits"].double() - ref).abs() <= tol).all())
        check_sample(s["token"], s["logits"], u, temperature=0.8, top_k=50, top_p=0.9)


def test_decode_step_captured(rt):
    step = Step(rt)
    k0, v0 = step.k.clone(), step.v.clone()
    eager = []
    for n in range(4):
        s = step(*step_inputs(n))
        eager.append({name: t.clone() for name, t in s.items()})
    step.k.copy_(k0)
    step.v.copy_(v0)
    static = step_inputs(0)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(*static)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s = step(*static)
    step.k.copy_(k0)
    step.v.copy_(v0)
    for n in range(4):
        for a, b in zip(static, step_inputs(n)):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        for name in s:
            assert torch.equal(s[name], eager[n][name]), (n, name)


# ------------------------------------------------- captures, streams, outputs
def q4_call(rt, seed=0):
    x, q, s, z = q4_inputs(3, 700, 1024, 64, "bfloat16", True, seed)
    return compiled(rt, graphs.matvec_q4(3, 700, 1024, 64, zeros=True), "bfloat16"), [x, q, s, z]


def rope_call(rt, seed=0):
    g = gen_of(seed)
    x = torch.randn(2, 9, 5, 64, generator=g, device=DEV).bfloat16()
    pos = torch.randint(0, 50, (3, 2, 9), generator=g, device=DEV, dtype=torch.int32)
    ck = compiled(rt, graphs.rope_positions(2, 9, 5, 64, table=50, sections=[16, 8, 8]), "bfloat16")
    return ck, [x, *tables(50, 32, seed), pos]


def few_call(rt, seed=0):
    q, k, v = attention_inputs(1, 1, 40000, 8, 1, 128, "bfloat16", seed)
    n = torch.tensor([39000 + seed], dtype=torch.int32, device=DEV)
    ck = window_kernel(rt, 1, 1, 40000, 8, 1, 128, None, 0, "bfloat16")
    assert ck.kernel.plan.kernels[0].config["parts"] > 1               # a workspace and a second kernel
    return ck, [q, k, v, n]


def tiles_call(rt, seed=0):
    q, k, v = attention_inputs(2, 100, 300, 8, 2, 64, "float16", seed)
    n = torch.tensor([300, 120 + seed], dtype=torch.int32, device=DEV)
    ck = window_kernel(rt, 2, 100, 300, 8, 2, 64, 70, 3, "float16")
    assert ck.kernel.plan.kernels[0].config["parts"] == 1
    return ck, [q, k, v, n]


def sample_call(rt, seed=0):
    x, u = sample_inputs(5, 30011, "float32", seed)
    ck = compiled(rt, graphs.sample(5, 30011, top_k=True, top_p=0.95), "float32")
    t = torch.full((5,), 0.9, device=DEV)
    return ck, [x, u, t, torch.tensor([0, 1, 50, 3000 + seed, 10], dtype=torch.int32, device=DEV)]


def parts_call(rt, seed=0):
    q, k, v = attention_inputs(1, 70, 2000, 4, 1, 128, "bfloat16", seed)
    n = torch.tensor([1900 + seed], dtype=torch.int32, device=DEV)
    ck = window_kernel(rt, 1, 70, 2000, 4, 1, 128, 1500, 3, "bfloat16")
    assert ck.kernel.plan.kernels[0].config["parts"] > 1
    return ck, [q, k, v, n]


CALLS = [q4_call, rope_call, few_call, tiles_call, parts_call, sample_call]


@pytest.mark.parametrize("call", CALLS)
def test_captured_and_replayed(rt, call):
    ck, ins = call(rt, 0)
    _, other = call(rt, 1)
    want = [ck(*ins).clone(), ck(*other).clone()]
    assert not torch.equal(*want)
    static = [t.clone() for t in ins]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ck(*static)
    for turn in (0, 1, 0):
        for a, b in zip(static, (ins, other)[turn]):
            a.copy_(b)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[turn])


@pytest.mark.parametrize("call", CALLS)
def test_two_captured_graphs_at_once(rt, call):
    ck, a = call(rt, 0)
    _, b = call(rt, 1)
    want = [ck(*a).clone(), ck(*b).clone()]
    runs = []
    for ins in (a, b):
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph, stream=side):
            out = [ck(*ins) for _ in range(8)]
        runs.append((graph, side, out))
    for _ in range(3):
        for graph, side, out in runs:
            with torch.cuda.stream(side):
                for o in out:
                    o.zero_()
                graph.replay()
        torch.cuda.synchronize()
        for (_, _, out), w in zip(runs, want):
            assert all(torch.equal(o, w) for o in out)


@pytest.mark.parametrize("call", CALLS)
def test_streams_and_given_outputs(rt, call):
    ck, ins = call(rt, 0)
    want = ck(*ins).clone()
    # inputs that the stream fills late: a call on another stream would read zeros
    for explicit in (False, True):
        late = [torch.zeros_like(t) for t in ins]
        out = torch.zeros_like(want)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)
            for t, s in zip(late, ins):
                t.copy_(s)
            if not explicit:
                got = ck(*late)
        if explicit:
            got = ck(*late, out=out, stream=side.cuda_stream)
            assert got is out or got.data_ptr() == out.data_ptr()
        side.synchronize()
        assert torch.equal(got, want)
    with pytest.raises(RuntimeError):
        ck(*ins, out=torch.empty(want.shape + (2,), dtype=want.dtype, device=DEV))


@pytest.mark.parametrize("call", CALLS)
def test_two_calls_at_once(rt, call):
    ck, a = call(rt, 0)
    _, b = call(rt, 1)
    want = [ck(*a).clone(), ck(*b).clone()]
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for j, ins in enumerate((a, b)):
            with torch.cuda.stream(sides[j]):
                got[j].append(ck(*ins))
    torch.cuda.synchronize()
    for j in (0, 1):
        assert all(torch.equal(o, want[j]) for o in got[j])


@pytest.mark.parametrize("call", CALLS)
def test_misaligned_and_strided_inputs(rt, call):
    ck, ins = call(rt, 0)
    want = ck(*ins).clone()
    for j, t in enumerate(ins):
        # the same values in every second element of a buffer
        wide = torch.zeros(t.shape + (2,), dtype=t.dtype, device=DEV)
        wide[..., 0] = t
        assert torch.equal(ck(*ins[:j], wide[..., 0], *ins[j + 1:]), want), j
    assert torch.equal(ck(*ins), want)


@pytest.mark.parametrize("first", ["exp", "product"])
def test_an_input_of_two_kernels_may_be_strided(rt, first):
    """Only the product takes rows with gaps; the other kernel of the graph
    needs x without them, whichever comes first."""
    g = DataflowGraph("both")
    x = g.add_input("x", TS([3, 256]), dtype="bfloat16")
    q = g.add_input("q", TS([64, 128]), dtype="uint8")
    s = g.add_input("s", TS([64, 4]), dtype="bfloat16")
    ops = {"exp": lambda: g.exp(x, "e"), "product": lambda: g.matvec_q4(x, q, s, name="y")}
    made = {name: ops[name]() for name in (("exp", "product") if first == "exp" else ("product", "exp"))}
    g.add_output(made["exp"])
    g.add_output(made["product"])
    xs, qs, ss, _ = q4_inputs(3, 64, 256, 64, "bfloat16", False)
    wide = torch.zeros(3, 512, dtype=torch.bfloat16, device=DEV)
    wide[:, :256] = xs
    e, y = Step.chain((g, [rt.compile(k) for k in compile_graph(g, dtype="bfloat16")]), wide[:, :256], qs, ss)
    check_q4(y, xs, qs, ss, None, "bfloat16")
    ref = torch.exp(xs.double())
    assert bool(((e.double() - ref).abs() <= (half_step("bfloat16") + 2.0 ** -20) * ref).all())


@pytest.mark.parametrize("call", CALLS)
def test_the_default_stream_by_number(rt, call):
    ck, ins = call(rt, 0)
    want = ck(*ins).clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ck(*ins, stream=torch.cuda.default_stream().cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_wrong_types_and_devices_are_refused(rt):
    ck, (q, k, v, n) = tiles_call(rt)
    with pytest.raises((RuntimeError, ValueError)):
        ck(q, k, v, n.long())
    with pytest.raises((RuntimeError, ValueError)):
        ck(q, k, v.float(), n)
    with pytest.raises(RuntimeError):
        ck(q, k, v, n.cpu())
    ck, (x, u, t, top_k) = sample_call(rt)
    with pytest.raises((RuntimeError, ValueError)):
        ck(x, u.double(), t, top_k)
    with pytest.raises((RuntimeError, ValueError)):
        ck(x, u[:-1], t, top_k)


@pytest.mark.parametrize("call,which", [(q4_call, [0]), (rope_call, [0]), (few_call, [0, 3]), (tiles_call, [0, 3]),
                                        (sample_call, [0, 1, 2, 3])])
def test_misplaced_inputs(rt, call, which):
    ck, ins = call(rt, 0)
    want = ck(*ins).clone()
    for j in which:
        buf = torch.empty(ins[j].numel() + 1, dtype=ins[j].dtype, device=DEV)
        moved = buf[1:].view(ins[j].shape)
        moved.copy_(ins[j])
        assert torch.equal(ck(*ins[:j], moved, *ins[j + 1:]), want), j


def test_misplaced_caches_are_refused(rt):
    for call in (few_call, tiles_call):
        ck, (q, k, v, n) = call(rt, 0)
        moved = torch.empty(k.numel() + 1, dtype=k.dtype, device=DEV)[1:].view(k.shape)
        for ins in ((q, moved, v, n), (q, k, moved, n)):
            with pytest.raises(_capi.MoltenError, match="aligned"):
                ck(*ins)


def test_outputs_do_not_overlap_inputs(rt):
    x, q, s, _ = q4_inputs(2, 256, 256, 64, "bfloat16", False)
    ck = compiled(rt, graphs.matvec_q4(2, 256, 256, 64), "bfloat16")
    with pytest.raises(RuntimeError, match="overlaps"):
        ck(x, q, s, out=x)
    ck, (qq, k, v, n) = tiles_call(rt)
    with pytest.raises(RuntimeError, match="overlaps"):
        ck(qq, k, v, n, out=qq)
    buf = torch.zeros(2 * qq.numel() - 8, dtype=qq.dtype, device=DEV)
    with pytest.raises(RuntimeError, match="overlaps"):
        ck(buf[:qq.numel()].view(qq.shape), k, v, n, out=buf[-qq.numel():].view(qq.shape))
    # RoPE in place
    ck, ins = rope_call(rt)
    want = ck(*ins).clone()
    assert ck(*ins, out=ins[0]).data_ptr() == ins[0].data_ptr() and torch.equal(ins[0], want)
    with pytest.raises(RuntimeError, match="overlaps"):
        wide = torch.zeros(want.numel() + 8, dtype=want.dtype, device=DEV)
        ck(wide[:-8].view(want.shape), *ins[1:], out=wide[8:].view(want.shape))


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_an_infinity_in_x_stays_in_its_row(rt, dtype):
    x, q, s, z = q4_inputs(4, 80, 512, 64, dtype, True)
    x[1, 100], x[2, 7] = torch.inf, torch.nan
    y = compiled(rt, graphs.matvec_q4(4, 80, 512, 64, zeros=True, dtype=dtype), dtype)(x, q, s, z)
    keep = torch.tensor([0, 3], device=DEV)
    check_q4(y[keep], x[keep], q, s, z, dtype)
    assert not torch.isfinite(y[1:3]).any()


@pytest.mark.parametrize("call", CALLS)
def test_short_ways_agree(rt, call):
    """The native short way, the same steps in Python and the general path."""
    from molten_b200.decode_launch import ModelCall, native_call
    assert native_call() is not None                 # (built with the rest of the library)
    ck, ins = call(rt, 0)
    want = ck(*ins).clone()
    spec = ck._spec_for(ins)
    assert isinstance(ck._last, ModelCall if call in (few_call, parts_call) else native_call())   # (parts: a second kernel)
    assert torch.equal(ModelCall(spec, ins)(tuple(ins)), want)
    assert torch.equal(ck._last(tuple(ins)), want)
    assert torch.equal(ck(*ins, out=torch.empty_like(want)), want)
    wide = torch.zeros(ins[0].shape + (2,), dtype=ins[0].dtype, device=DEV)[..., 0]
    for other in (tuple(ins[:-1]), (wide, *ins[1:]), (ins[0].float(), *ins[1:]) if ins[0].dtype != torch.float32
                  else (ins[0].half(), *ins[1:]), (ins[0][:1], *ins[1:]), (ins[0].cpu(), *ins[1:])):
        if other[0].shape != ins[0].shape or other[0].dtype != ins[0].dtype or other[0] is wide or len(other) < len(ins) \
                or not other[0].is_cuda:
            assert ck._last(other) is NotImplemented


def test_short_way_of_one_token_attention(rt):
    q, k, v = attention_inputs(2, 1, 300, 8, 2, 128, "bfloat16")
    n = torch.tensor([300, 77], dtype=torch.int32, device=DEV)
    for lengths in (True, False):
        ck = window_kernel(rt, 2, 1, 300, 8, 2, 128, 100, 2, "bfloat16", lengths=lengths)
        ins = (q, k, v, n) if lengths else (q, k, v)
        for _ in range(3):
            check_attention(ck(*ins), q, k, v, n if lengths else torch.full_like(n, 300), 100, 2, "bfloat16", 2.0 ** -16)


def test_shapes_in_turn(rt):
    ck = compiled(rt, graphs.sample(4, 1000), "float32")
    cases = [(sample_inputs(r, v, "float32", r), torch.full((r,), 1.3, device=DEV))
             for r, v in ((4, 1000), (1, 77), (9, 20001))]
    want = [ck(x, u, t).clone() for (x, u), t in cases]
    for _ in range(3):
        for ((x, u), t), w in zip(cases, want):
            assert torch.equal(ck(x, u, t), w)
    for ((x, u), t), w in zip(cases, want):
        check_sample(w, x, u, temperature=t)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("top_p", [None, 0.6])
@pytest.mark.parametrize("top_k", [None, 21])        # (0.6 of 21 equal weights ends inside one)
def test_sample_extreme_temperatures(rt, dtype, top_p, top_k):
    x, u = sample_inputs(8, 3001, dtype, seed=5)
    x[:, 7] = -torch.inf
    x[:, 9] = torch.nan
    t = torch.tensor([1e-3, 1e-20, 1e-31, 0.0, -1.0, 50.0, 1e30, torch.inf], device=DEV)
    given = {k: v for k, v in (("top_p", top_p), ("top_k", top_k)) if v is not None}
    tokens = compiled(rt, graphs.sample(8, 3001, dtype=dtype, **given), dtype)(x, u, t)
    # with a temperature past all logits every kept token weighs the same
    check_sample(tokens[:-2], x[:-2], u[:-2], temperature=t[:-2].where(t[:-2] >= 1e-30, 0.0), **given)
    check_sample(tokens[-2:], x[-2:], u[-2:], temperature=torch.tensor([1e30, 1e300], dtype=torch.float64), **given)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,vocab,top_p", [(64, 131072, 0.93), (64, 131072, 0.999), (40, 20011, 0.99)])
def test_sample_many_kept_tokens(rt, dtype, rows, vocab, top_p):
    """Flat rows, of which the filters keep more or fewer tokens than fit the
    packed list."""
    x, u = sample_inputs(rows, vocab, dtype, seed=rows)
    t = torch.linspace(0.5, 3.0, rows, device=DEV)
    tokens = compiled(rt, graphs.sample(rows, vocab, dtype=dtype, top_p=top_p), dtype)(x, u, t)
    check_sample(tokens, x, u, temperature=t, top_p=torch.full((rows,), top_p))


# ---------------------------------------------------- tensors that coincide
def test_the_same_tensor_twice(rt):
    x, q, s, _ = q4_inputs(2, 100, 256, 64, "bfloat16", False)
    ck = compiled(rt, graphs.matvec_q4(2, 100, 256, 64, zeros=True), "bfloat16")
    for _ in range(2):
        check_q4(ck(x, q, s, s), x, q, s, s, "bfloat16")
    for new in (1, 50):
        qq, k, _ = attention_inputs(2, new, 90, 4, 2, 64, "bfloat16", new)
        n = torch.tensor([90, 60], dtype=torch.int32, device=DEV)
        att = window_kernel(rt, 2, new, 90, 4, 2, 64, 20, 1, "bfloat16")
        check_attention(att(qq, k, k, n), qq, k, k, n, 20, 1, "bfloat16", 2.0 ** -8)
        # and queries from the same buffer (each key head twice)
        qs = k[:, -new:].repeat_interleave(2, 2)
        check_attention(att(qs, k, k, n), qs, k, k, n, 20, 1, "bfloat16", 2.0 ** -8)
    cos, _ = tables(40, 16)
    xr = torch.randn(1, 7, 3, 32, generator=gen_of(1), device=DEV)
    pos = torch.arange(7, dtype=torch.int32, device=DEV).view(1, 1, 7)
    rope = compiled(rt, graphs.rope_positions(1, 7, 3, 32, table=40, dtype="float32"), "float32")
    check_rope(rope(xr, cos, cos, pos), xr, cos, cos, pos, [16], "half", "float32")
    lg, u = sample_inputs(6, 501, "float32")
    pick = compiled(rt, graphs.sample(6, 501, top_p=True), "float32")
    check_sample(pick(lg, u, u, u), lg, u, temperature=u, top_p=u)


def test_one_graph_input_in_two_places(rt):
    g = DataflowGraph("shared")
    q = g.add_input("q", TS([1, 3, 4, 64]), dtype="bfloat16")
    k = g.add_input("k", TS([1, 30, 2, 64]), dtype="bfloat16")
    g.add_output(g.window_attention(q, k, k, window=10, sinks=1))
    ck = compiled(rt, g, "bfloat16")
    qq, kk, _ = attention_inputs(1, 3, 30, 4, 2, 64, "bfloat16")
    n = torch.tensor([30], dtype=torch.int32, device=DEV)
    for _ in range(2):
        check_attention(ck(qq, kk), qq, kk, kk, n, 10, 1, "bfloat16", 2.0 ** -16)


# -------------------------------------------------------------- empty batches
def test_empty_batches(rt):
    x, q, s, z = q4_inputs(1, 64, 256, 64, "bfloat16", True)
    assert compiled(rt, graphs.matvec_q4(1, 64, 256, 64, zeros=True), "bfloat16")(x[:0], q, s, z).shape == (0, 64)
    for new in (1, 40):
        qq, k, v = attention_inputs(1, new, 50, 4, 2, 64, "bfloat16")
        n = torch.tensor([50], dtype=torch.int32, device=DEV)
        ck = window_kernel(rt, 1, new, 50, 4, 2, 64, 20, 1, "bfloat16")
        assert ck(qq[:0], k[:0], v[:0], n[:0]).shape == (0, new, 4, 64)
    lg, u = sample_inputs(3, 100, "float32")
    t = torch.ones(3, device=DEV)
    assert compiled(rt, graphs.sample(3, 100), "float32")(lg[:0], u[:0], t[:0]).shape == (0,)
    cos, sin = tables(8, 16)
    ck = compiled(rt, graphs.rope_positions(1, 4, 2, 32, table=8), "bfloat16")
    pos = torch.zeros(1, 1, 0, dtype=torch.int32, device=DEV)
    assert ck(torch.empty(1, 0, 2, 32, dtype=torch.bfloat16, device=DEV), cos, sin, pos).shape == (1, 0, 2, 32)


# ------------------------------------------------------- past 2^31 elements
def test_long_cache(rt):
    cache, kv, d, window, sinks = 2 ** 21 + 1000, 8, 128, 300, 4
    k = torch.zeros(1, cache, kv, d, dtype=torch.bfloat16, device=DEV)
    v = torch.zeros(1, cache, kv, d, dtype=torch.bfloat16, device=DEV)
    assert k.numel() > 2 ** 31
    g = gen_of(3)
    for t in (k, v):
        t[:, :sinks] = torch.randn(1, sinks, kv, d, generator=g, device=DEV)
        t[:, -1500:] = torch.randn(1, 1500, kv, d, generator=g, device=DEV)
    for new, length in ((1, cache), (1, cache - 7), (200, cache - 1)):
        q = torch.randn(1, new, kv * 2, d, generator=g, device=DEV).bfloat16()
        n = torch.tensor([length], dtype=torch.int32, device=DEV)
        out = window_kernel(rt, 1, new, cache, kv * 2, kv, d, window, sinks, "bfloat16")(q, k, v, n)
        # the same attention over a cache without the middle
        cut = cache - 1500 - sinks
        ks, vs = (torch.cat((t[:, :sinks], t[:, -1500:]), 1) for t in (k, v))
        check_attention(out, q, ks, vs, n - cut, window, sinks, "bfloat16", 2.0 ** -8)


def test_many_weights(rt):
    n, k = 1_100_000, 4096
    q = torch.zeros(n, k // 2, dtype=torch.uint8, device=DEV)
    assert q.numel() > 2 ** 31
    x, qt, s, _ = q4_inputs(2, 500, k, 128, "bfloat16", False)
    q[-500:] = qt
    scales = torch.full((n, k // 128), 0.01, dtype=torch.bfloat16, device=DEV)
    scales[-500:] = s
    y = compiled(rt, graphs.matvec_q4(2, n, k, 128), "bfloat16")(x, q, scales)
    check_q4(y[:, -500:], x, qt, s, None, "bfloat16")
    check_q4(y[:, :500], x, q[:500], scales[:500], None, "bfloat16")


def test_many_logits(rt):
    rows, vocab = 17000, 131072
    x = torch.zeros(rows, vocab, dtype=torch.bfloat16, device=DEV)
    assert x.numel() > 2 ** 31
    few, u = sample_inputs(20, vocab, "bfloat16")
    x[-20:] = few
    us = torch.full((rows,), 0.5, device=DEV)
    us[-20:] = u
    t = torch.ones(rows, device=DEV)
    tokens = compiled(rt, graphs.sample(rows, vocab, dtype="bfloat16", top_p=0.7), "bfloat16")(x, us, t)
    check_sample(tokens[-20:], few, u, top_p=0.7)
    # equal logits: the first 91751 reach 0.7f of all; half of those is 45875.5
    assert (tokens[:-20] == 45875).all()


def test_many_tokens(rt):
    seq, heads, d = 2 ** 18 + 5, 64, 128
    x = torch.zeros(1, seq, heads, d, dtype=torch.bfloat16, device=DEV)
    assert x.numel() > 2 ** 31
    x[:, -3:] = torch.randn(1, 3, heads, d, generator=gen_of(1), device=DEV)
    cos, sin = tables(100, d // 2)
    pos = torch.randint(0, 100, (1, 1, seq), generator=gen_of(2), device=DEV, dtype=torch.int32)
    out = compiled(rt, graphs.rope_positions(1, seq, heads, d, table=100), "bfloat16")(x, cos, sin, pos)
    check_rope(out[:, -3:], x[:, -3:], cos, sin, pos[..., -3:], [d // 2], "half", "bfloat16")
    assert not out[:, :-3].any()


# ------------------------------------------------------ calls on a named stream
@pytest.mark.parametrize("call", CALLS)
def test_strided_inputs_on_a_named_stream(rt, call):
    """Copies of strided inputs are made on the stream of the call, which fills
    them late; on the current one they would hold zeros."""
    ck, ins = call(rt, 0)
    want = ck(*ins).clone()
    wide = [torch.zeros(t.shape + (2,), dtype=t.dtype, device=DEV) for t in ins]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        for w, t in zip(wide, ins):
            w[..., 0].copy_(t)
    got = ck(*(w[..., 0] for w in wide), stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(got, want)


def test_outputs_of_a_named_stream_take_no_memory_in_use(rt):
    """Memory that was freed while the current stream still reads it is not an
    output of another stream, and an output that the current stream reads is not
    taken again by the other one."""
    x, q, s, z = q4_inputs(32, 16384, 512, 64, "float32", True)
    ck = compiled(rt, graphs.matvec_q4(32, 16384, 512, 64, zeros=True, dtype="float32"), "float32")
    want = ck(x, q, s, z).clone()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        old = torch.full_like(want, 7.0)
        torch.cuda._sleep(20_000_000)
        kept = old + 1.0
        del old
        got = ck(x, q, s, z, stream=side.cuda_stream)
        torch.cuda.synchronize()
        assert bool((kept == 8.0).all()) and torch.equal(got, want)
        del got, kept
        got = ck(x, q, s, z, stream=side.cuda_stream)
        side.synchronize()
        torch.cuda._sleep(20_000_000)
        kept = got + 1.0
        del got
        with torch.cuda.stream(side):
            torch.full_like(want, 7.0)
        torch.cuda.synchronize()
        assert torch.equal(kept, want + 1.0)
        del kept


# ------------------------------------------------------- the first call captured
def fresh(tmp_path, call):
    """``call`` with a runtime whose modules are not loaded yet."""
    import shutil
    ck, _ = call(MoltenRuntime(), 0)
    (tmp_path / "cache").mkdir()
    shutil.copy(ck._module, tmp_path / "cache")
    return call(MoltenRuntime(cache_dir=str(tmp_path / "cache")), 0)


@pytest.mark.parametrize("call", CALLS)
def test_the_first_call_may_be_captured(rt, call, tmp_path):
    """Modules are loaded by the first call, also where that is recorded."""
    want = call(rt, 0)[0](*call(rt, 0)[1]).clone()
    ck, ins = fresh(tmp_path, call)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ck(*ins)
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


@pytest.mark.parametrize("call", CALLS)
def test_a_compiled_kernel_is_ready(rt, call, monkeypatch):
    """compile() loads the module and makes the short way: the first call with
    the declared shapes does neither, and builds no parameter block by itself."""
    from molten_b200 import runtime
    torch.zeros(1, device=DEV)
    ck, ins = call(MoltenRuntime(), 0)
    assert ck._last is not None
    monkeypatch.setattr(runtime, "loaded_module", None)
    monkeypatch.setattr(runtime, "short_call", None)
    monkeypatch.setattr(type(ck), "_spec_for", None)
    assert torch.equal(ck(*ins), call(rt, 0)[0](*ins))


def test_the_first_call_of_other_families_may_be_captured(tmp_path):
    g = graphs.rmsnorm(64, 512, dtype="bfloat16")
    x = torch.randn(64, 512, generator=gen_of(1), device=DEV).bfloat16()
    w = torch.ones(512, device=DEV).bfloat16()
    k = compile_graph(g, dtype="bfloat16")[0]
    want = MoltenRuntime().compile(k)(x, w)
    ck = MoltenRuntime(cache_dir=str(tmp_path)).compile(k)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ck(x, w)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_the_first_call_of_a_process_may_be_captured():
    """The status word is allocated with the first kernel that has one."""
    import subprocess
    import sys
    from pathlib import Path
    code = """
import torch
from tests.test_decode_step_gpu import rope_call, tiles_call
from molten_b200.runtime import MoltenRuntime
rt = MoltenRuntime()
for call in (rope_call, tiles_call):
    ck, ins = call(rt, 0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ck(*ins)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, ck(*ins))
assert MoltenRuntime.read_status(0) == 0
"""
    done = subprocess.run([sys.executable, "-c", code], cwd=Path(__file__).parents[1], capture_output=True, text=True,
                          timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


# ----------------------------------------------------------- cost of a call
@pytest.mark.parametrize("call", CALLS)
def test_the_short_way_is_made_once(call, monkeypatch):
    """Calls that cannot take it (a given output or stream, strided inputs, other
    shapes in turn) do not make it again."""
    from molten_b200 import runtime
    made = []
    short_call = runtime.short_call
    monkeypatch.setattr(runtime, "short_call", lambda *args: made.append(args) or short_call(*args))
    ck, ins = call(MoltenRuntime(), 0)
    want = ck(*ins).clone()
    out = torch.empty_like(want)
    wide = torch.zeros(ins[0].shape + (2,), dtype=ins[0].dtype, device=DEV)
    wide[..., 0] = ins[0]
    for _ in range(4):
        assert torch.equal(ck(*ins, out=out), want)
        assert torch.equal(ck(*ins, stream=torch.cuda.current_stream().cuda_stream), want)
        assert torch.equal(ck(wide[..., 0], *ins[1:]), want)
        assert torch.equal(ck(*ins), want)
    assert len(made) == 1


@pytest.mark.parametrize("call", CALLS)
def test_a_named_stream_inside_a_capture(rt, call):
    """A branch of a recorded graph: the call's stream follows the captured one
    and is joined again."""
    ck, ins = call(rt, 0)
    want = ck(*ins).clone()
    wide = torch.zeros(ins[0].shape + (2,), dtype=ins[0].dtype, device=DEV)
    wide[..., 0] = ins[0]
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        here = torch.cuda.current_stream()
        side.wait_stream(here)
        out = ck(wide[..., 0], *ins[1:], stream=side.cuda_stream)
        here.wait_stream(side)
        copy = out.clone()
        del out
    for _ in range(3):
        copy.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(copy, want)


@pytest.mark.parametrize("call", CALLS)
def test_outputs_stay_inside_their_memory(rt, call):
    ck, ins = call(rt, 0)
    want, guard = ck(*ins).clone(), 2048
    kept = [t.clone() for t in ins]
    bits = {2: torch.int16, 4: torch.int32}[want.element_size()]
    buf = torch.randint(-1000, 1000, (want.numel() + 2 * guard,), generator=gen_of(71), device=DEV, dtype=bits)
    before = buf.clone()
    out = buf[guard:-guard].view(want.dtype).view(want.shape)
    ck(*ins, out=out)
    assert torch.equal(out, want)
    assert torch.equal(buf[:guard], before[:guard]) and torch.equal(buf[-guard:], before[-guard:])
    assert all(torch.equal(a, b) for a, b in zip(ins, kept))


@pytest.mark.parametrize("d", [8, 24, 72, 104])
@pytest.mark.parametrize("new,heads,kv", [(1, 5, 1), (3, 6, 2), (60, 7, 1), (130, 6, 2)])
def test_odd_head_dims_stay_inside_their_memory(rt, d, new, heads, kv):
    b, cache = 2, 150
    q, k, v = attention_inputs(b, new, cache, heads, kv, d, "bfloat16", d)
    n = torch.tensor([150, 131], dtype=torch.int32, device=DEV)
    ck = window_kernel(rt, b, new, cache, heads, kv, d, 40, 2, "bfloat16")
    buf = torch.full((q.numel() + 4096,), 7.0, dtype=torch.bfloat16, device=DEV)
    out = buf[2048:-2048].view(q.shape)
    ck(q, k, v, n, out=out)
    check_attention(out, q, k, v, n, 40, 2, "bfloat16", half_step("bfloat16"))
    assert bool((buf[:2048] == 7.0).all()) and bool((buf[-2048:] == 7.0).all())
