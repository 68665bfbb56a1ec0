"""The operators of a decode step on a B200, against plain 64-bit forms."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from molten_b200 import _capi, graphs
from molten_b200.codegen import compile_graph
from molten_b200.ir import DataflowGraph, TensorShape as TS
from molten_b200.lowering import LoweringError
from molten_b200.runtime import MoltenRuntime

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
DT = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


@pytest.fixture(scope="module")
def rt():
    return MoltenRuntime()


def gen_of(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def compiled(rt, g, dtype):
    ks = compile_graph(g, dtype=dtype)
    assert len(ks) == 1
    return rt.compile(ks[0])


def half_step(dtype):
    return torch.finfo(DT[dtype]).eps / 2


# ------------------------------------------------------------- 4-bit products
def q4_inputs(m, n, k, group, dtype, zeros, seed=0):
    g = gen_of(seed)
    x = torch.randn(m, k, generator=g, device=DEV).to(DT[dtype])
    q = torch.randint(0, 256, (n, k // 2), generator=g, device=DEV, dtype=torch.uint8)
    s = ((0.5 + torch.rand(n, k // group, generator=g, device=DEV)) / k ** 0.5).to(DT[dtype])
    z = (16 * torch.rand(n, k // group, generator=g, device=DEV)).to(DT[dtype]) if zeros else None
    return x, q, s, z


def q4_reference(x, q, s, z):
    """(y, sum of |terms|) in 64 bits."""
    n, k = q.shape[0], q.shape[1] * 2
    w = torch.stack((q & 15, q >> 4), -1).view(n, s.shape[1], -1).double()
    zp = z.double()[:, :, None] if z is not None else 8.0
    sd = s.double()[:, :, None]
    mag = ((w - 8).abs() + (zp - 8.0 if z is None else (zp - 8.0).abs())) * sd
    w = ((w - zp) * sd).view(n, k)
    return x.double() @ w.t(), x.double().abs() @ mag.view(n, k).t()


def check_q4(y, x, q, s, z, dtype):
    ref, mag = q4_reference(x, q, s, z)
    # one output rounding; at most 24 MMAs a group, each off by at most one
    # step (2^-23) of the magnitudes it sums, and the fp32 sum over groups
    tol = half_step(dtype) * ref.abs() + 2.0 ** -18 * mag
    err = (y.double() - ref).abs()
    assert bool((err <= tol).all()), f"max error {err.max().item():.3e}"
    # the errors are not systematic: the fp32 result as a whole is near
    if dtype == "float32":
        assert err.norm() <= 1e-6 * ref.norm()


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("m,n,k,group", [
    (1, 1, 32, 32), (1, 16, 128, 128), (1, 17, 64, 64), (2, 33, 96, 32), (3, 100, 192, 64),
    (8, 257, 1152, 128), (9, 48, 4096, 32), (16, 640, 512, 64), (17, 31, 2176, 128),
    (32, 1000, 1024, 32), (5, 4099, 160, 32)])
def test_matvec_q4(rt, m, n, k, group, dtype, zeros):
    x, q, s, z = q4_inputs(m, n, k, group, dtype, zeros, seed=m + n)
    ck = compiled(rt, graphs.matvec_q4(m, n, k, group, dtype=dtype, zeros=zeros), dtype)
    args = [x, q, s] + ([z] if zeros else [])
    y = ck(*args)
    assert y.shape == (m, n) and y.dtype == DT[dtype]
    check_q4(y, x, q, s, z, dtype)
    assert torch.equal(y, ck(*args))


@pytest.mark.parametrize("warps,warps_n,ksplit", [
    (8, 1, 1), (8, 1, 8), (8, 2, 2), (16, 4, 4), (8, 8, 1), (16, 8, 8), (16, 16, 1), (16, 1, 2)])
def test_matvec_q4_splits(rt, warps, warps_n, ksplit):
    m, n, k, group = 4, 200, 8192, 128
    tuned = MoltenRuntime(tune={"q4": {"warps": warps, "warps_n": warps_n, "ksplit": ksplit}})
    ck = compiled(tuned, graphs.matvec_q4(m, n, k, group, zeros=True), "bfloat16")
    # (another shape than the declared one: the runtime's tune applies)
    x2, q2, s2, z2 = q4_inputs(m, n + 1, k, group, "bfloat16", True, seed=4)
    check_q4(ck(x2, q2, s2, z2), x2, q2, s2, z2, "bfloat16")


@pytest.mark.parametrize("m,n,k,group,dtype", [
    (32, 700, 14336, 32, "bfloat16"), (20, 3000, 5120, 64, "float32"), (2, 40000, 256, 128, "float16"),
    (1, 5000, 60000 // 32 * 32, 32, "float32"), (7, 130, 32768, 128, "bfloat16")])
def test_matvec_q4_chunks_and_many_tiles(rt, m, n, k, group, dtype):
    """x staged in several chunks of k; CTAs that walk over many tiles."""
    x, q, s, z = q4_inputs(m, n, k, group, dtype, True, seed=5)
    ck = compiled(rt, graphs.matvec_q4(m, n, k, group, dtype=dtype, zeros=True), dtype)
    check_q4(ck(x, q, s, z), x, q, s, z, dtype)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_matvec_q4_range_of_x(rt, dtype):
    """Rows and groups of very different size, zeros, and the largest values."""
    m, n, k, group = 5, 64, 512, 64
    x, q, s, z = q4_inputs(m, n, k, group, dtype, True, seed=6)
    power = torch.tensor([0, 100, -100, 60, -60, 20, 119, -10], device=DEV).repeat_interleave(group)
    x = (x.double() * torch.exp2(power.double())).to(DT[dtype])
    x[1] = 0
    x[2, ::2] = 0
    x[3, :group] *= 2.0 ** -30
    ck = compiled(rt, graphs.matvec_q4(m, n, k, group, dtype=dtype, zeros=True), dtype)
    check_q4(ck(x, q, s, z), x, q, s, z, dtype)


def test_matvec_q4_mixed_types_rank_and_strides(rt):
    """bf16 x with fp32 scales, x [2, 2, K] out of a wider tensor."""
    k, n, group = 256, 70, 64
    _, q, s, z = q4_inputs(1, n, k, group, "float32", True, seed=5)
    wide = torch.randn(2, 2, 3 * k, generator=gen_of(6), device=DEV).to(torch.bfloat16)
    x = wide[..., k:2 * k]
    g = DataflowGraph("q4")
    ids = [g.add_input("x", TS([2, 2, k])), g.add_input("q", TS([n, k // 2]), dtype="uint8"),
           g.add_input("s", TS([n, k // group]), dtype="float32"),
           g.add_input("z", TS([n, k // group]), dtype="float32")]
    g.add_output(g.matvec_q4(ids[0], ids[1], ids[2], zeros=ids[3]))
    ck = compiled(rt, g, "bfloat16")
    y = ck(x, q, s, z)
    assert y.shape == (2, 2, n)
    check_q4(y.view(4, n), x.reshape(4, k), q, s, z, "bfloat16")


def test_matvec_q4_in_a_group(rt):
    """RMSNorm -> 4-bit product -> + bias -> SiLU as one graph."""
    m, n, k, group = 4, 192, 512, 128
    x, q, s, _ = q4_inputs(m, n, k, group, "bfloat16", False, seed=7)
    w = (1 + 0.1 * torch.randn(k, generator=gen_of(8), device=DEV)).to(torch.bfloat16)
    b = torch.randn(n, generator=gen_of(9), device=DEV).to(torch.bfloat16)
    g = DataflowGraph("norm_q4")
    xi, wi = g.add_input("x", TS([m, k])), g.add_input("w", TS([k]))
    qi = g.add_input("q", TS([n, k // 2]), dtype="uint8")
    si, bi = g.add_input("s", TS([n, k // group]), dtype="bfloat16"), g.add_input("b", TS([n]))
    y = g.matvec_q4(g.rms_norm(xi, wi, "norm"), qi, si)
    g.add_output(g.silu(g.add(y, bi)))
    out = compiled(rt, g, "bfloat16")(x, w, q, s, b)
    xd = x.double()
    h = xd / (xd.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
    ref, _ = q4_reference(h, q, s, None)
    _, mag = q4_reference(h, q, s, None)
    ref = ref + b.double()
    # the normalised rows are rounded to bf16 once, the result once; SiLU's
    # slope is at most 1.1
    tol = 2.0 ** -8 * 1.1 * mag + 2.0 ** -8 * ref.abs() + 1e-4
    assert bool(((out.double() - torch.nn.functional.silu(ref)).abs() <= tol).all())


def test_matvec_q4_refuses_unaligned_pointers(rt):
    x, q, s, _ = q4_inputs(1, 16, 128, 128, "bfloat16", False)
    ck = compiled(rt, graphs.matvec_q4(1, 16, 128, 128), "bfloat16")
    raw = torch.empty(16 * 64 + 1, dtype=torch.uint8, device=DEV)
    with pytest.raises(_capi.MoltenError, match="aligned"):
        ck(x, raw[1:].view(16, 64), s)
    with pytest.raises(LoweringError):
        ck(x.float().int(), q, s)


# ------------------------------------------------------ rotary at positions
def rope_reference(x, cos, sin, pos, sections, style):
    half = x.shape[-1] // 2
    axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections)).to(DEV)
    rows = pos.long().view(len(sections), *x.shape[:-2])[axis].movedim(0, -1)     # [.., seq, pair]
    pair = torch.arange(half, device=DEV)
    pad = rows < 0
    c = cos.double()[rows.clamp(min=0), pair].masked_fill(pad, 1.0)[..., None, :]
    s = sin.double()[rows.clamp(min=0), pair].masked_fill(pad, 0.0)[..., None, :]
    xd = x.double()
    a, b = (xd[..., :half], xd[..., half:]) if style == "half" else (xd[..., 0::2], xd[..., 1::2])
    r0, r1 = a * c - b * s, a * s + b * c
    mag = (a * c).abs() + (b * s).abs() + (a * s).abs() + (b * c).abs()
    if style == "half":
        return torch.cat((r0, r1), -1), torch.cat((mag, mag), -1)
    return torch.stack((r0, r1), -1).flatten(-2), torch.stack((mag, mag), -1).flatten(-2)


def check_rope(out, x, cos, sin, pos, sections, style, dtype):
    ref, mag = rope_reference(x, cos, sin, pos, sections, style)
    # one rounding; two fp32 products and a sum before it
    tol = half_step(dtype) * ref.abs() + 2 * 2.0 ** -24 * mag + 2.0 ** -24 * ref.abs()
    assert bool(((out.double() - ref).abs() <= tol).all())


def tables(rows, half, seed=1, dtype=torch.float32):
    a = torch.rand(rows, half, generator=gen_of(seed), device=DEV, dtype=torch.float64) * 6.3
    return torch.cos(a).to(dtype), torch.sin(a).to(dtype)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("style", ["half", "interleaved"])
@pytest.mark.parametrize("batch,seq,heads,dim,sections", [
    (1, 1, 1, 2, [1]), (3, 1, 40, 128, [64]), (2, 5, 7, 128, [16, 24, 24]), (1, 33, 4, 80, [13, 27]),
    (2, 9, 3, 6, [1, 1, 1]), (1, 300, 5, 96, [0, 48]), (1, 4, 2, 64, [5, 7, 9, 11]),
    (1, 3, 2, 1024, [512])])
def test_rope_positions(rt, batch, seq, heads, dim, sections, style, dtype):
    rows = 57
    x = torch.randn(batch, seq, heads, dim, generator=gen_of(2), device=DEV).to(DT[dtype])
    cos, sin = tables(rows, dim // 2)
    pos = torch.randint(-2, rows, (len(sections), batch, seq), generator=gen_of(3), device=DEV,
                        dtype=torch.int32)
    g = graphs.rope_positions(batch, seq, heads, dim, rows, sections, dtype=dtype, style=style)
    out = compiled(rt, g, dtype)(x, cos, sin, pos)
    check_rope(out, x, cos, sin, pos, sections, style, dtype)
    assert MoltenRuntime.read_status(0) == 0
    # padding: both halves of a pair are left bit for bit
    skip = (pos < 0).all(0)
    assert torch.equal(out[skip], x[skip])


@pytest.mark.parametrize("style", ["half", "interleaved"])
def test_rope_positions_many_heads_per_thread(rt, style):
    """Many tokens, more heads than a CTA takes at once."""
    x = torch.randn(2, 4700, 22, 128, generator=gen_of(2), device=DEV).to(torch.bfloat16)
    cos, sin = tables(4096, 64)
    pos = torch.randint(0, 4096, (2, 4700), generator=gen_of(3), device=DEV, dtype=torch.int32)
    ck = compiled(rt, graphs.rope_positions(2, 4700, 22, 128, 4096, style=style), "bfloat16")
    check_rope(ck(x, cos, sin, pos), x, cos, sin, pos, [64], style, "bfloat16")


def test_rope_positions_views_tables_and_alignment(rt):
    """x out of a fused q, k, v tensor; 16-bit and packed tables; pointers
    that are not 16-byte aligned."""
    b, s, h, d, rows = 2, 6, 3, 64, 40
    fused = torch.randn(b, s, 3 * h, d, generator=gen_of(4), device=DEV).to(torch.float16)
    x = fused[:, :, h:2 * h]
    cos, sin = tables(rows, d // 2, dtype=torch.bfloat16)
    pos = torch.randint(0, rows, (b, s), generator=gen_of(5), device=DEV, dtype=torch.int32)
    ck = compiled(rt, graphs.rope_positions(b, s, h, d, rows, dtype="float16",
                                            table_dtype="bfloat16"), "float16")
    check_rope(ck(x, cos, sin, pos), x, cos, sin, pos, [32], "half", "float16")
    packed = torch.stack((cos, sin), -1).flatten(1).float()
    g = graphs.rope_positions(b, s, h, d, rows, dtype="float16", packed=True, style="interleaved")
    check_rope(compiled(rt, g, "float16")(x, packed, pos), x, cos, sin, pos, [32], "interleaved",
               "float16")
    odd = torch.empty(x.numel() + 1, dtype=torch.float16, device=DEV)[1:].view(x.shape)
    odd.copy_(x)
    check_rope(ck(odd, cos, sin, pos), x, cos, sin, pos, [32], "half", "float16")


def test_rope_position_past_the_table_is_reported(rt):
    x = torch.randn(1, 3, 2, 8, generator=gen_of(6), device=DEV)
    cos, sin = tables(5, 4)
    pos = torch.tensor([[0, 5, 4]], dtype=torch.int32, device=DEV)
    out = compiled(rt, graphs.rope_positions(1, 3, 2, 8, 5, dtype="float32"), "float32")(x, cos, sin, pos)
    assert torch.equal(out[:, 1], x[:, 1])
    assert MoltenRuntime.read_status(0) == 4096 and MoltenRuntime.read_status(0) == 0


# --------------------------------------------------------- window attention
def seen_mask(lengths, new, cache, window, sinks):
    """[batch, new, cache]: query i sees key j."""
    n = lengths.long().clamp(0, cache)[:, None, None]
    p = n - new + torch.arange(new, device=DEV)[:, None]
    j = torch.arange(cache, device=DEV)
    near = torch.ones_like(j, dtype=torch.bool) if window is None else (j > p - window) | (j < sinks)
    return (j <= p) & (j < n) & near


def attention_reference(q, k, v, lengths, window, sinks, scale=None):
    """(o, sum p |v|, largest |score|) in 64 bits; unseen keys are left out."""
    b, new, heads, d = q.shape
    cache, kv = k.shape[1:3]
    scale = d ** -0.5 if scale is None else scale
    seen = seen_mask(lengths, new, cache, window, sinks)[:, None, None]            # b 1 1 new cache
    used = seen.any(3)[:, 0, 0]                                                    # b cache
    kd = torch.where(used[:, :, None, None], k.double(), 0.0)
    vd = torch.where(used[:, :, None, None], v.double(), 0.0)
    qd = q.double().view(b, new, kv, heads // kv, d)
    s = torch.einsum("bnkgd,bckd->bkgnc", qd, kd) * scale
    s = torch.where(seen, s, -torch.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.where(seen, torch.exp(s - torch.where(top == -torch.inf, 0.0, top)), 0.0)
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
    o = torch.einsum("bkgnc,bckd->bnkgd", p, vd)
    mag = torch.einsum("bkgnc,bckd->bnkgd", p, vd.abs())
    big = torch.where(seen, s, 0.0).abs().amax(-1)                                  # b kv per new
    big = big.permute(0, 3, 1, 2)[..., None]
    return (t.expand(b, new, kv, heads // kv, d).reshape(b, new, heads, d) for t in (o, mag, big))


def check_attention(out, q, k, v, lengths, window, sinks, dtype, p_half, scale=None):
    ref, mag, big = attention_reference(q, k, v, lengths, window, sinks, scale)
    # one output rounding; P rounded to `p_half` of itself; scores summed in
    # fp32 (d products, 2^-23 each of the largest score, and the exponential's
    # argument again) and exponentials within 2^-20, in P and in its sum
    tol = half_step(dtype) * ref.abs() + (p_half + 2.0 ** -19 + 2.0 ** -21 * (1 + big)) * mag
    # subnormal outputs and weights of fp16
    tol = tol + (2.0 ** -24 if dtype == "float16" else 0.0)
    err = (out.double() - ref).abs()
    assert bool((err <= tol).all()), f"max error {err.max().item():.3e}"


def attention_inputs(b, new, cache, heads, kv, d, dtype, seed=0, spread=1.0):
    g = gen_of(seed)
    q = (spread * torch.randn(b, new, heads, d, generator=g, device=DEV)).to(DT[dtype])
    k = torch.randn(b, cache, kv, d, generator=g, device=DEV).to(DT[dtype])
    v = torch.randn(b, cache, kv, d, generator=g, device=DEV).to(DT[dtype])
    return q, k, v


def window_kernel(rt, b, new, cache, heads, kv, d, window, sinks, dtype, lengths=True, scale=None):
    g = graphs.window_attention(b, new, cache, heads, kv, d, window=window, sinks=sinks, dtype=dtype,
                                lengths=lengths, scale=scale)
    return compiled(rt, g, dtype)


FEW = [  # b, new, cache, heads, kv, d, window, sinks, lengths
    (1, 1, 1, 1, 1, 64, 1, 0, [1]),
    (3, 1, 40, 4, 2, 64, 7, 2, [40, 3, 0]),
    (2, 1, 300, 8, 2, 128, 100, 4, [300, 150]),
    (2, 1, 1000, 12, 4, 80, None, 0, [1000, 999]),
    (4, 1, 515, 16, 1, 128, 64, 33, [515, 64, 65, 17]),
    (2, 2, 130, 10, 2, 8, 16, 1, [130, 1]),
    (1, 4, 2500, 32, 8, 128, 1024, 16, [2333]),
    (2, 3, 77, 20, 2, 96, 30, 0, [77, 2]),
    (1, 32, 200, 4, 4, 64, 50, 5, [180]),
    (5, 1, 33, 7, 7, 24, 1, 3, [33, 32, 31, 5, -4]),
    (1, 1, 9000, 8, 1, 128, None, 0, [9001]),
]


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("case", FEW)
def test_window_attention_few_rows(rt, case, dtype):
    b, new, cache, heads, kv, d, window, sinks, lens = case
    q, k, v = attention_inputs(b, new, cache, heads, kv, d, dtype, seed=cache)
    lengths = torch.tensor(lens, dtype=torch.int32, device=DEV)
    ck = window_kernel(rt, b, new, cache, heads, kv, d, window, sinks, dtype)
    out = ck(q, k, v, lengths)
    assert out.shape == q.shape and out.dtype == q.dtype
    check_attention(out, q, k, v, lengths, window, sinks, dtype, 2.0 ** -16)
    assert torch.equal(out, ck(q, k, v, lengths))


@pytest.mark.parametrize("ranks,parts", [(1, 1), (2, 1), (8, 1), (1, 3), (4, 5), (8, 7)])
def test_window_attention_splits(ranks, parts):
    """Clusters and parts, with requests shorter than the split."""
    b, new, cache, heads, kv, d = 3, 2, 700, 8, 2, 64
    tuned = MoltenRuntime(tune={"window": {"ranks": ranks, "parts": parts}})
    ck = window_kernel(tuned, 1, 1, 16, heads, kv, d, 300, 4, "bfloat16")
    q, k, v = attention_inputs(b, new, cache, heads, kv, d, "bfloat16", seed=1)
    lengths = torch.tensor([700, 20, 0], dtype=torch.int32, device=DEV)
    check_attention(ck(q, k, v, lengths), q, k, v, lengths, 300, 4, "bfloat16", 2.0 ** -16)


@pytest.mark.parametrize("new", [1, 3])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), torch.finfo(torch.bfloat16).min])
def test_window_attention_ignores_unseen_keys(rt, new, bad):
    """Whatever stands behind a request's length, before its window, or ahead
    of a query does not reach it."""
    b, cache, heads, kv, d, window, sinks = 2, 120, 8, 2, 64, 40, 3
    q, k, v = attention_inputs(b, new, cache, heads, kv, d, "bfloat16", seed=2)
    lengths = torch.tensor([97, 60], dtype=torch.int32, device=DEV)
    seen = seen_mask(lengths, new, cache, window, sinks)
    unseen = ~seen.any(1)
    k[unseen], v[unseen] = bad, bad
    ck = window_kernel(rt, b, new, cache, heads, kv, d, window, sinks, "bfloat16")
    out = ck(q, k, v, lengths)
    check_attention(out, q, k, v, lengths, window, sinks, "bfloat16", 2.0 ** -16)
    if new > 1:
        # the newest value: only the last query may notice
        v2 = v.clone()
        v2[torch.arange(b, device=DEV), lengths.long() - 1] = bad
        got = ck(q, k, v2, lengths)
        # (the same sums in another order for the rows that share the tile)
        check_attention(got[:, :-1], q[:, :-1], k, v, lengths - 1, window, sinks, "bfloat16", 2.0 ** -16)
        if bad != bad or bad == float("inf"):
            assert not bool(torch.isfinite(got[:, -1]).any())


def test_window_attention_views_and_scale(rt):
    """q, k, v out of one fused tensor; caches laid out [batch, heads, seq, d];
    a given scale; large scores."""
    b, new, heads, kv, d, cache = 2, 2, 8, 4, 64, 90
    fused = torch.randn(b, new, heads + 2 * kv, d, generator=gen_of(3), device=DEV).to(torch.float16)
    q = fused[:, :, :heads] * 4
    kc = torch.randn(b, kv, cache + 6, d, generator=gen_of(4), device=DEV).to(torch.float16)
    vc = torch.randn(b, kv, cache + 6, d, generator=gen_of(5), device=DEV).to(torch.float16)
    k, v = kc[:, :, 6:].transpose(1, 2), vc[:, :, 6:].transpose(1, 2)
    lengths = torch.tensor([90, 31], dtype=torch.int32, device=DEV)
    ck = window_kernel(rt, b, new, cache, heads, kv, d, 25, 1, "float16", scale=1.5)
    out = ck(fused[:, :, :heads] * 4, k, v, lengths)
    check_attention(out, q, k, v, lengths, 25, 1, "float16", 2.0 ** -16, scale=1.5)
    full = torch.full((b,), cache, dtype=torch.int32, device=DEV)
    none = window_kernel(rt, b, new, cache, heads, kv, d, None, 0, "float16", lengths=False)
    check_attention(none(q, k, v), q, k, v, full, None, 0, "float16", 2.0 ** -16)


MANY = [  # b, new, cache, heads, kv, d, window, sinks, lengths
    (1, 40, 40, 2, 2, 64, None, 0, [40]),
    (1, 128, 128, 1, 1, 128, None, 0, [128]),
    (1, 257, 257, 1, 1, 64, 100, 3, [257]),
    (2, 300, 300, 4, 2, 128, 128, 4, [300, 170]),
    (2, 130, 900, 8, 2, 128, 200, 130, [900, 411]),
    (1, 700, 1500, 5, 1, 80, 333, 16, [1500]),
    (3, 65, 400, 14, 2, 96, 1, 0, [400, 65, 30]),
    (2, 90, 500, 8, 8, 24, 50, 1, [0, 499]),
    (1, 2000, 2000, 2, 1, 128, 512, 129, [2000]),
    (1, 33, 3000, 128, 1, 64, 700, 5, [2999]),
    (2, 600, 700, 6, 2, 128, 2000, 0, [700, 644]),
]


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("case", MANY)
def test_window_attention_many_rows(rt, case, dtype):
    b, new, cache, heads, kv, d, window, sinks, lens = case
    q, k, v = attention_inputs(b, new, cache, heads, kv, d, dtype, seed=cache + new)
    lengths = torch.tensor(lens, dtype=torch.int32, device=DEV)
    ck = window_kernel(rt, b, new, cache, heads, kv, d, window, sinks, dtype)
    assert ck.specialization(q, k, v, lengths).plan.kernels[0].config["kind"] == "tiles"
    out = ck(q, k, v, lengths)
    assert MoltenRuntime.read_status(0) == 0
    check_attention(out, q, k, v, lengths, window, sinks, dtype, half_step(dtype))
    assert torch.equal(out, ck(q, k, v, lengths))


@pytest.mark.parametrize("parts", [1, 2, 3, 7, 32])
@pytest.mark.parametrize("case", [
    (1, 40, 1000, 8, 2, 128, 300, 5, [1000]), (2, 90, 700, 6, 2, 64, None, 0, [700, 40]),
    (1, 300, 2000, 4, 4, 80, 130, 200, [1900]), (3, 65, 300, 7, 1, 128, 17, 1, [300, 0, 66])])
def test_window_attention_many_rows_in_parts(parts, case):
    """CTAs that share the key tiles of an item; some see no key of some Q tile."""
    b, new, cache, heads, kv, d, window, sinks, lens = case
    q, k, v = attention_inputs(b, new, cache, heads, kv, d, "bfloat16", seed=cache)
    lengths = torch.tensor(lens, dtype=torch.int32, device=DEV)
    # (compiled for other sizes: the call's plan takes the given parts)
    ck = window_kernel(MoltenRuntime(tune={"window": {"parts": parts}}), 1, 130, 140, heads, kv, d, window, sinks,
                       "bfloat16")
    out = ck(q, k, v, lengths)
    assert ck.specialization(q, k, v, lengths).plan.kernels[0].config["parts"] == parts
    check_attention(out, q, k, v, lengths, window, sinks, "bfloat16", 2.0 ** -8)
    assert torch.equal(ck(q, k, v, lengths), out)
    # an infinity of V that some queries see, and one behind the lengths
    v = v.clone()
    v[0, lens[0] - 2, 0, 3] = torch.inf
    v[:, max(lens):] = torch.nan
    bad = ck(q, k, v, lengths)
    seen = seen_mask(lengths, new, cache, window, sinks)[0, :, lens[0] - 2]
    per = heads // kv
    assert (bad[0, seen][:, :per, 3] == torch.inf).all()
    keep = torch.ones_like(out, dtype=torch.bool)
    keep[0, :, :per, 3] = ~seen[:, None]
    assert torch.equal(bad[keep], out[keep])


@pytest.mark.parametrize("spread", [8.0, 60.0])
def test_window_attention_growing_maxima(rt, spread):
    """Scores whose maxima grow along the keys: O is rescaled, and large
    differences leave single keys."""
    b, new, cache, heads, kv, d = 1, 200, 1200, 4, 2, 64
    q, k, v = attention_inputs(b, new, cache, heads, kv, d, "bfloat16", seed=7, spread=spread)
    k = (k * torch.linspace(0.05, 1.0, cache, device=DEV)[None, :, None, None]).to(torch.bfloat16)
    lengths = torch.tensor([cache], dtype=torch.int32, device=DEV)
    ck = window_kernel(rt, b, new, cache, heads, kv, d, None, 0, "bfloat16")
    out = ck(q, k, v, lengths)
    check_attention(out, q, k, v, lengths, None, 0, "bfloat16", 2.0 ** -8)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), torch.finfo(torch.bfloat16).min])
def test_window_attention_many_rows_ignores_unseen_keys(rt, bad):
    b, new, cache, heads, kv, d, window, sinks = 2, 150, 900, 4, 2, 128, 130, 3
    q, k, v = attention_inputs(b, new, cache, heads, kv, d, "bfloat16", seed=8)
    lengths = torch.tensor([811, 120], dtype=torch.int32, device=DEV)
    unseen = ~seen_mask(lengths, new, cache, window, sinks).any(1)
    k[unseen], v[unseen] = bad, bad
    ck = window_kernel(rt, b, new, cache, heads, kv, d, window, sinks, "bfloat16")
    check_attention(ck(q, k, v, lengths), q, k, v, lengths, window, sinks, "bfloat16", 2.0 ** -8)
    if bad != bad or bad == float("inf"):
        # one value that only the last 10 queries see, one that only the first do
        v2 = v.clone()
        v2[0, 801, 0, 5] = bad
        v2[0, 811 - 150 - 100, 1, 7] = bad
        got = ck(q, k, v2, lengths)
        v2[0, 801, 0, 5] = 0
        v2[0, 811 - 150 - 100, 1, 7] = 0
        ref, _, _ = attention_reference(q, k, v2, lengths, window, sinks)
        seen = seen_mask(lengths, new, cache, window, sinks)[0]
        hit = torch.zeros_like(got, dtype=torch.bool)
        hit[0, :, :2, 5] = seen[:, 801][:, None]
        hit[0, :, 2:, 7] = seen[:, 811 - 150 - 100][:, None]
        assert int(hit.sum()) > 0 and torch.equal(~torch.isfinite(got), hit)
        assert bool(((got.double() - ref).abs() <= 0.05)[~hit].all())


def test_window_attention_many_rows_views(rt):
    b, new, heads, kv, d, cache = 2, 100, 8, 4, 64, 333
    fused = torch.randn(b, new, heads + 2 * kv, d, generator=gen_of(3), device=DEV).to(torch.float16)
    q = fused[:, :, :heads]
    kc = torch.randn(b, kv, cache + 6, d, generator=gen_of(4), device=DEV).to(torch.float16)
    vc = torch.randn(1, cache, kv, d, generator=gen_of(5), device=DEV).to(torch.float16)
    k, v = kc[:, :, 6:].transpose(1, 2), vc.expand(b, cache, kv, d)
    lengths = torch.tensor([cache, 131], dtype=torch.int32, device=DEV)
    ck = window_kernel(rt, b, new, cache, heads, kv, d, 90, 1, "float16", scale=0.3)
    check_attention(ck(q, k, v, lengths), q, k, v, lengths, 90, 1, "float16", 2.0 ** -11, scale=0.3)
    # the same through the few-row kernel's form of the parameters: one row at a time
    one = window_kernel(rt, b, 1, cache, heads, kv, d, 90, 1, "float16", scale=0.3)
    got = one(q[:, -1:], k, v, lengths)
    check_attention(got, q[:, -1:], k, v, lengths, 90, 1, "float16", 2.0 ** -16, scale=0.3)


# ------------------------------------------------------------------ sampling
def sample_reference(logits, u, temperature=None, top_k=None, top_p=None, min_p=None):
    """(tokens, how near any border came to a decision), in 64 bits."""
    x_all = logits.double().cpu().numpy()
    rows = x_all.shape[0]

    def of(v, r, none):
        return none if v is None else float(v[r]) if torch.is_tensor(v) else float(v)
    out, near = np.empty(rows, np.int64), np.empty(rows)
    for r in range(rows):
        x = np.where(np.isnan(x_all[r]), -np.inf, np.minimum(x_all[r], 3.4028234663852886e38))
        t, k, p, mp = of(temperature, r, 1.0), of(top_k, r, 0), of(top_p, r, 1.0), of(min_p, r, 0.0)
        order = np.argsort(-x, kind="stable")
        near[r] = 1.0
        if x[order[0]] == -np.inf:
            out[r] = -1
            continue
        if not t > 0:
            out[r] = order[0]
            continue
        count = int(np.sum(x > -np.inf))
        if k > 0:
            count = min(count, int(k))
        w = np.exp((x[order[:count]] - x[order[0]]) / t)
        if p < 1:
            reach = np.cumsum(w)
            goal = max(p, 0.0) * reach[-1]
            near[r] = min(near[r], np.min(np.abs(reach / reach[-1] - p)) if p > 0 else 1.0)
            count = max(1, int(np.searchsorted(reach, goal, side="left")) + (1 if goal > 0 else 0))
            count = min(count, w.size)
        if mp > 0:
            near[r] = min(near[r], np.min(np.abs(w[:count] - mp)))
            count = max(1, int(np.sum(w[:count] >= min(mp, 1.0))))
        chosen = np.sort(order[:count])
        reach = np.cumsum(np.exp((x[chosen] - x[order[0]]) / t))
        goal = float(u[r]) * reach[-1]
        near[r] = min(near[r], np.min(np.abs(reach - goal)) / reach[-1])
        out[r] = chosen[min(np.searchsorted(reach, goal, side="right"), chosen.size - 1)]
    return out, near


def check_sample(tokens, logits, u, **params):
    want, near = sample_reference(logits, u, **params)
    got = tokens.cpu().numpy()
    # where a border lies within 1e-10 of the decision, 64 bits do not decide it
    sure = near > 1e-10
    assert sure.mean() > 0.9
    assert np.array_equal(got[sure], want[sure]), np.flatnonzero((got != want) & sure)[:8]


def sample_inputs(rows, vocab, dtype, seed=0, spread=3.0):
    g = gen_of(seed)
    x = (spread * torch.randn(rows, vocab, generator=g, device=DEV)).to(DT[dtype])
    return x, torch.rand(rows, generator=g, device=DEV)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (5, 2), (3, 7), (40, 300), (33, 5003), (9, 50257), (4, 131072)])
@pytest.mark.parametrize("use", ["", "k", "p", "m", "kp", "kpm"])
def test_sample(rt, rows, vocab, dtype, use):
    x, u = sample_inputs(rows, vocab, dtype, seed=rows + vocab)
    g = gen_of(9)
    params = {"temperature": 0.3 + 1.5 * torch.rand(rows, generator=g, device=DEV)}
    if "k" in use:
        params["top_k"] = torch.randint(-1, min(vocab + 2, 3000), (rows,), generator=g, device=DEV,
                                        dtype=torch.int32)
    if "p" in use:
        params["top_p"] = 1.1 * torch.rand(rows, generator=g, device=DEV)
    if "m" in use:
        params["min_p"] = 0.3 * torch.rand(rows, generator=g, device=DEV) - 0.05
    ck = compiled(rt, graphs.sample(rows, vocab, dtype=dtype, top_k="k" in use, top_p="p" in use,
                                    min_p="m" in use), dtype)
    tokens = ck(x, u, *params.values())
    assert tokens.dtype == torch.int32 and tokens.shape == (rows,)
    check_sample(tokens, x, u, **params)
    assert torch.equal(tokens, ck(x, u, *params.values()))


@pytest.mark.parametrize("ranks", [1, 2, 4, 8])
@pytest.mark.parametrize("kind", ["ties", "equal", "steps", "narrow", "wide", "one"])
def test_sample_hard_rows(ranks, kind):
    """Rows whose borders fall into many equal logits, spread over 40 orders of
    magnitude or lie a rounding apart."""
    rows, vocab = 24, 20011
    tuned = MoltenRuntime(tune={"sample": {"ranks": ranks}})
    ck = compiled(tuned, graphs.sample(2, 64, top_k=True, top_p=True, min_p=True), "float32")
    g = gen_of(11)
    x = torch.randn(rows, vocab, generator=g, device=DEV)
    if kind == "ties":
        x = (4 * x).round() / 2
    elif kind == "equal":
        x = torch.full_like(x, 3.25)
    elif kind == "steps":
        x = torch.arange(vocab, device=DEV).float().expand(rows, vocab) % 97 * 0.01
    elif kind == "narrow":
        x = 1000 + x * 1e-4
    elif kind == "wide":
        x = x * torch.exp(20 * torch.rand(rows, vocab, generator=g, device=DEV) - 10) * 1e30
    else:
        x = torch.full_like(x, -torch.inf)
        x[torch.arange(rows, device=DEV), torch.randint(0, vocab, (rows,), generator=g, device=DEV)] = 2.0
    x = x.contiguous()
    u = torch.rand(rows, generator=g, device=DEV)
    params = {"temperature": 0.5 + torch.rand(rows, generator=g, device=DEV),
              "top_k": torch.randint(0, vocab, (rows,), generator=g, device=DEV, dtype=torch.int32),
              "top_p": 0.3 + 0.8 * torch.rand(rows, generator=g, device=DEV),
              "min_p": 0.1 * torch.rand(rows, generator=g, device=DEV) - 0.05}
    if kind == "wide":
        params["temperature"] *= 1e33
    check_sample(ck(x, u, *params.values()), x, u, **params)


def test_sample_edges(rt):
    """Greedy rows, rows without a token, infinities and NaN, u at its ends,
    parameters that keep only the largest token."""
    vocab = 1000
    inf, nan = float("inf"), float("nan")
    base = torch.randn(12, vocab, generator=gen_of(12), device=DEV)
    x = base.clone()
    x[0] = -inf
    x[1] = nan
    x[2, 5::7] = nan
    x[3, 100], x[3, 200] = inf, inf
    x[4, 17], x[4, 9] = 9.0, 9.0
    x[5, :-1] = -inf
    u = torch.tensor([.3, .3, .5, .7, .9, .5, 0., 1 - 2.0 ** -24, .5, .5, .5, .5], device=DEV)
    t = torch.tensor([1, 1, 1, 1, 0, 1, 1, 1, -1, 1e-6, 1e30, 1], device=DEV)
    k = torch.tensor([0, 5, 50, 0, 3, 2, 0, 0, 1, 0, 0, 1], dtype=torch.int32, device=DEV)
    p = torch.tensor([.5, .5, .9, .99, .1, .5, 1, 1, 1, 1, .5, 0.], device=DEV)
    m = torch.tensor([0, 0, 0, 0, 0, .5, 0, 0, 0, 0, 0, 2.], device=DEV)
    ck = compiled(rt, graphs.sample(12, vocab, top_k=True, top_p=True, min_p=True), "float32")
    tokens = ck(x, u, t, k, p, m)
    check_sample(tokens, x, u, temperature=t, top_k=k, top_p=p, min_p=m)
    assert tokens[0] == -1 and tokens[1] == -1 and tokens[4] == 9 and tokens[5] == vocab - 1
    assert tokens[3] in (100, 200)


def test_sample_constants_views_and_rank(rt):
    """Scalar parameters, a strided view, two leading dims."""
    wide = 2 * torch.randn(3, 4, 777, generator=gen_of(13), device=DEV).to(torch.bfloat16)
    x = wide[..., 5:506]
    u = torch.rand(3, 4, generator=gen_of(14), device=DEV)
    g = DataflowGraph("sample")
    xi, ui = g.add_input("x", TS([3, 4, 501])), g.add_input("u", TS([3, 4]))
    g.add_output(g.sample(xi, ui, temperature=g.add_constant("t", 0.7), top_k=g.add_constant("k", 40),
                          top_p=g.add_constant("p", 0.8)))
    tokens = compiled(rt, g, "bfloat16")(x, u)
    assert tokens.shape == (3, 4)
    check_sample(tokens.view(12), x.reshape(12, 501), u.view(12), temperature=0.7, top_k=40, top_p=0.8)
    # greedy
    g = DataflowGraph("greedy")
    xi, ui = g.add_input("x", TS([3, 4, 501])), g.add_input("u", TS([3, 4]))
    g.add_output(g.sample(xi, ui, temperature=g.add_constant("t", 0.0)))
    assert torch.equal(compiled(rt, g, "bfloat16")(x, u).long().view(12),
                       torch.from_numpy(sample_reference(x.reshape(12, 501), u.view(12), 0.0)[0]).to(DEV))


@pytest.mark.parametrize("vocab", [1, 3, 700, 3000])
def test_sample_ranks_without_tokens(vocab):
    """Clusters of 8 CTAs, most of which hold no token and reach the first
    exchange at once; many more rows than run at a time."""
    rows = 3000
    ck = compiled(MoltenRuntime(tune={"sample": {"ranks": 8}}), graphs.sample(2, 64, top_k=True, top_p=0.9), "float32")
    x, u = sample_inputs(rows, vocab, "float32", seed=vocab)
    t = torch.ones(rows, device=DEV)
    k = torch.full((rows,), 40, dtype=torch.int32, device=DEV)
    tokens = ck(x, u, t, k)
    assert ck.specialization(x, u, t, k).plan.kernels[0].config["ranks"] == 8
    check_sample(tokens[:200], x[:200], u[:200], top_k=k, top_p=0.9)
    for _ in range(20):
        assert torch.equal(ck(x, u, t, k), tokens)


@pytest.mark.parametrize("top", [10.0, -10.0, 1000.0])
@pytest.mark.parametrize("use", ["", "k", "p", "m"])
def test_sample_temperatures_below_the_spacing_of_logits(rt, top, use):
    """The largest fp32 logit twice behind one 1 to 20 steps below it, with
    temperatures from a thousandth of a step to some 30 of them: the lower one
    weighs something, nothing, or less than any number."""
    vocab, steps = 20000, 20
    spacing = float(np.spacing(np.float32(top)))
    ts = spacing * 2.0 ** torch.linspace(-11, 5, 48, device=DEV)
    rows = steps * ts.numel()
    x = top - 100 - 5 * torch.rand(rows, vocab, generator=gen_of(21), device=DEV)
    at = torch.randint(1, vocab - 1, (rows,), generator=gen_of(22), device=DEV)
    ups = torch.arange(1, steps + 1, device=DEV).repeat_interleave(ts.numel())
    row = torch.arange(rows, device=DEV)
    x[row, at - 1] = (top - ups.double() * spacing).float()            # (exact)
    x[row, at], x[row, at + 1] = top, top
    u = torch.rand(rows, generator=gen_of(23), device=DEV)
    params = {"temperature": ts.repeat(steps)}
    if use == "k":
        params["top_k"] = torch.full((rows,), 4, dtype=torch.int32, device=DEV)
    elif use:
        params["top_p" if use == "p" else "min_p"] = torch.full((rows,), 0.97 if use == "p" else 1e-3, device=DEV)
    ck = compiled(rt, graphs.sample(rows, vocab, top_k=use == "k", top_p=use == "p", min_p=use == "m"), "float32")
    out = torch.full((rows,), -7, dtype=torch.int32, device=DEV)
    ck(x, u, *params.values(), out=out)
    check_sample(out, x, u, **params)


@pytest.mark.parametrize("kind", ["infinite", "cold", "hot"])
def test_sample_masks_of_the_lowest_value(rt, kind):
    """Masks of the type's lowest value beside +inf (the largest value), under
    very low and under infinite temperatures: differences of two logits pass
    the type's range."""
    rows, vocab = 16, 3001
    x, u = sample_inputs(rows, vocab, "float32", seed=31)
    x[:, 5::3] = torch.finfo(torch.float32).min
    t = 0.4 + torch.rand(rows, generator=gen_of(32), device=DEV)
    if kind == "cold":
        x[:, 7::500] = 9.0                             # (six of them)
        t = 10.0 ** torch.linspace(-9, -28, rows, device=DEV)
    else:
        x[:, 7::500] = torch.inf
    if kind == "hot":
        t = torch.full_like(t, torch.inf)
        t[::2] = 10.0 ** torch.linspace(36, 38.4, rows // 2, device=DEV)
    for top_p in (0.55, 0.85):
        tokens = compiled(rt, graphs.sample(rows, vocab, top_p=top_p), "float32")(x, u, t)
        check_sample(tokens, x, u, temperature=t.double().clamp(max=1e300), top_p=top_p)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("new,cache,ranks,parts", [(1, 40, 1, 1), (1, 700, 8, 1), (1, 700, 2, 3), (4, 700, 1, 1),
                                                   (4, 700, 8, 2)])
def test_window_attention_few_rows_keeps_infinities(new, cache, ranks, parts, dtype):
    """An infinity in a value that a query sees is that infinity in its output;
    both of them, or a NaN, are NaN."""
    b, heads, kv, d, window, sinks = 2, 8, 2, 64, 300, 4
    rt = MoltenRuntime(tune={"window": {"ranks": ranks, "parts": parts}})
    ck = window_kernel(rt, 1, 1, 16, heads, kv, d, window, sinks, dtype)
    q, k, v = attention_inputs(b, new, cache, heads, kv, d, dtype, seed=3)
    lengths = torch.tensor([cache, cache - 9], dtype=torch.int32, device=DEV)
    clean = ck(q, k, v, lengths)
    n, per = cache - new - 2, heads // kv              # (a key that every query of request 0 sees)
    v[0, n, 0, 1], v[0, 2, 0, 2] = torch.inf, -torch.inf
    v[0, n, 0, 3], v[0, n - 1, 0, 3] = torch.inf, -torch.inf
    v[0, n, 0, 4] = torch.nan
    out = ck(q, k, v, lengths)
    assert bool((out[0, :, :per, 1] == torch.inf).all()) and bool((out[0, :, :per, 2] == -torch.inf).all())
    assert bool(torch.isnan(out[0, :, :per, 3:5]).all())
    keep = torch.ones_like(out, dtype=torch.bool)
    keep[0, :, :per, 1:5] = False
    assert bool(torch.isfinite(out[keep]).all())
    v[0, n - 1:n + 1, 0, 1:5], v[0, 2, 0, 2] = 0.0, 0.0
    ref, mag, big = attention_reference(q, k, v, lengths, window, sinks)
    # (check_attention's tolerance)
    tol = half_step(dtype) * ref.abs() + (2.0 ** -16 + 2.0 ** -19 + 2.0 ** -21 * (1 + big)) * mag + (
        2.0 ** -24 if dtype == "float16" else 0.0)
    assert bool(((out.double() - ref).abs() <= tol)[keep].all())
    assert torch.equal(out[1], clean[1])


@pytest.mark.parametrize("new,cache,d,parts", [(1, 300, 64, None), (3, 300, 128, None), (100, 300, 64, None),
                                               (90, 700, 80, 1), (90, 700, 24, 1), (300, 900, 128, 3)])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_window_attention_in_a_group(new, cache, d, parts, dtype):
    """Attention -> + residual -> SiLU as one graph: the attention is kept in
    32 bits between them."""
    b, heads, kv, window, sinks = 2, 6, 2, 150, 3
    g = DataflowGraph("attention_residual")
    ids = [g.add_input("q", TS([b, new, heads, d])), g.add_input("k", TS([b, cache, kv, d])),
           g.add_input("v", TS([b, cache, kv, d])), g.add_input("n", TS([b]), dtype="int32")]
    r = g.add_input("r", TS([b, new, heads, d]))
    g.add_output(g.silu(g.add(g.window_attention(*ids[:3], lengths=ids[3], window=window, sinks=sinks), r)))
    ck = MoltenRuntime(tune={"window": {"parts": parts}} if parts else {}).compile(compile_graph(g, dtype=dtype)[0])
    # (another batch than the declared one: planned with the given parts)
    q, kk, v = attention_inputs(b + 1, new, cache, heads, kv, d, dtype, seed=d)
    res = torch.randn(b + 1, new, heads, d, generator=gen_of(41), device=DEV).to(DT[dtype])
    lengths = torch.tensor([cache, new + 7, 0], dtype=torch.int32, device=DEV)
    v[0, cache - 1, 0, 3] = torch.inf                  # (the last query's alone)
    out = ck(q, kk, v, lengths, res)
    plan = ck.specialization(q, kk, v, lengths, res).plan
    assert [sk.outputs[0].dtype for sk in plan.kernels] == ["float32", dtype]
    bad = torch.zeros_like(out, dtype=torch.bool)
    bad[0, -1, :heads // kv, 3] = True
    assert bool((out[bad] == torch.inf).all())
    v[0, cache - 1, 0, 3] = 0.0
    ref, mag, big = attention_reference(q, kk, v, lengths, window, sinks)
    y = ref + res.double()
    # P's rounding, scores and exponentials as in check_attention, the sum in
    # fp32, SiLU's slope of at most 1.1 and one output rounding
    p_half = half_step(dtype) if plan.kernels[0].config["kind"] == "tiles" else 2.0 ** -16
    want = torch.nn.functional.silu(y)
    tol = (half_step(dtype) + 2.0 ** -20) * want.abs() + 1.1 * (
        (p_half + 2.0 ** -19 + 2.0 ** -21 * (1 + big)) * mag + 2.0 ** -23 * y.abs() + 2.0 ** -24)
    err = (out.double() - want).abs()
    assert bool((err <= tol)[~bad].all()), err[~bad].max().item()


@pytest.mark.parametrize("order", ["pcsx", "cxsp"])
@pytest.mark.parametrize("shape,style,dtype", [((3, 700, 22, 128), "half", "bfloat16"), ((1, 9, 3, 6), "interleaved", "float32")])
def test_rope_in_place_with_x_anywhere(rt, order, shape, style, dtype):
    b, s, h, d = shape
    g = DataflowGraph("turned")
    ids = {}
    for n in order:
        dims = {"x": shape, "c": (50, d // 2), "s": (50, d // 2), "p": (1, b, s)}[n]
        ids[n] = g.add_input(n, TS(list(dims)), dtype={"x": dtype, "p": "int32"}.get(n, "float32"))
    g.add_output(g.rope(ids["x"], ids["c"], sin=ids["s"], positions=ids["p"], style=style))
    ck = compiled(rt, g, dtype)
    cos, sin = tables(50, d // 2)
    x = torch.randn(*shape, generator=gen_of(1), device=DEV).to(DT[dtype])
    pos = torch.randint(-1, 50, (1, b, s), generator=gen_of(2), device=DEV, dtype=torch.int32)
    t = {"x": x, "c": cos, "s": sin, "p": pos}
    want = ck(*[t[n] for n in order])
    check_rope(want, x, cos, sin, pos, [d // 2], style, dtype)
    y = x.clone()
    ck(*[dict(t, x=y)[n] for n in order], out=y)
    assert torch.equal(y, want)
    over = torch.zeros(max(x.numel(), cos.numel()), device=DEV, dtype=torch.float32)
    wide = dict(t, c=over[:cos.numel()].view(cos.shape))
    with pytest.raises(RuntimeError, match="overlaps"):
        ck(*[wide[n] for n in order], out=over.view(DT[dtype])[:x.numel()].view(shape))


@pytest.mark.parametrize("gap", [1, 7, 8])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_window_attention_infinities_between_empty_requests(rt, gap, bad):
    """Requests of one key tile with an infinity, and between those of one CTA
    requests of length 0, which cost the warps that clean V nothing."""
    sms, new, heads, d = 148, 40, 1, 64
    turns = 3 * gap + 1
    b = sms * turns
    q, k, v = attention_inputs(b, new, new, heads, 1, d, "bfloat16", seed=5)
    full = torch.arange(b, device=DEV) // sms % gap == 0
    lengths = torch.where(full, new, 0).to(torch.int32)
    ck = window_kernel(rt, b, new, new, heads, 1, d, None, 0, "bfloat16")
    c = ck.kernel.plan.kernels[0].config
    assert c["kind"] == "tiles" and c["parts"] == 1 and c["items"] == b
    clean = ck(q, k, v, lengths)
    check_attention(clean, q, k, v, lengths, None, 0, "bfloat16", half_step("bfloat16"))
    at = 5 + torch.arange(b, device=DEV) % 30
    v[torch.arange(b, device=DEV), at, 0, 9] = bad
    for _ in range(5):
        out = ck(q, k, v, lengths)
        hit = full[:, None] & (torch.arange(new, device=DEV) >= at[:, None])
        got = out[:, :, 0, 9].float()
        assert bool((torch.isnan(got) if bad != bad else got == bad)[hit].all())
        assert bool(torch.isfinite(got[~hit]).all())
        others = torch.ones(d, dtype=torch.bool, device=DEV)
        others[9] = False
        assert torch.equal(out[..., others], clean[..., others])


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("m,n,k,group,tune", [
    (3, 80, 512, 64, {}), (9, 33, 4096, 128, {}), (20, 130, 1024, 32, {}), (5, 300, 8192, 128, {"ksplit": 8}),
    (32, 700, 14336, 32, {})])
def test_matvec_q4_infinities_in_x(m, n, k, group, tune, zeros, dtype):
    """An infinity in x makes every output of its row that infinity times the
    weight's sign, NaN where the weight is 0 or where signs meet."""
    x, q, s, z = q4_inputs(m, n, k, group, dtype, zeros, seed=11)
    if zeros:
        z = z.round()                                  # (weights of 0 among them)
    ck = compiled(MoltenRuntime(tune={"q4": tune}), graphs.matvec_q4(1, 16, group, group, dtype=dtype, zeros=zeros),
                  dtype)
    x[0, 5] = torch.inf
    x[1, k - 1] = -torch.inf
    x[2, 3], x[2, group + 1] = torch.inf, torch.inf
    rows = 3
    if m > 4:
        x[3, 7] = torch.nan
        x[4, 0], x[4, 9] = torch.inf, -torch.inf
        rows = 5
    y = ck(x, q, s, *([z] if zeros else []))
    w = (torch.stack((q & 15, q >> 4), -1).view(n, s.shape[1], -1).double()
         - (z.double()[:, :, None] if zeros else 8.0)) * s.double()[:, :, None]
    ref = torch.stack([(r.double() * w.view(n, k)).sum(1) for r in x[:rows]])
    assert torch.equal(torch.isnan(y[:rows]), torch.isnan(ref))
    signs = dict(nan=0.0, posinf=1.0, neginf=-1.0)
    assert torch.equal(y[:rows].double().nan_to_num(**signs), ref.nan_to_num(**signs))
    if m > rows:
        check_q4(y[rows:], x[rows:], q, s, z, dtype)


def test_matvec_q4_sums_past_the_range(rt):
    """Rows near the largest fp32 value, whose sums pass it, with weights that
    keep the product within it."""
    m, n, k, group = 4, 48, 512, 64
    _, q, s, z = q4_inputs(m, n, k, group, "float32", True, seed=13)
    x = 3e38 * (0.5 + 0.5 * torch.rand(m, k, generator=gen_of(14), device=DEV))
    s = s * 1e-6
    y = compiled(rt, graphs.matvec_q4(m, n, k, group, dtype="float32", zeros=True), "float32")(x, q, s, z)
    check_q4(y, x, q, s, z, "float32")


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("new,gap", [(1, 12.0), (1, 17.0), (4, 17.0), (100, 12.0), (100, 16.0)])
def test_window_attention_weights_far_below_the_largest(rt, new, gap, dtype):
    """A first key that takes nearly all the weight and has a value of 0, as
    sinks do: the output is what e^-12 to e^-17 of it leaves to 20000 others."""
    b, cache, heads, kv, d = 1, 20000, 4, 1, 64
    q, k, v = attention_inputs(b, new, cache, heads, kv, d, dtype, seed=9)
    k = 0.3 * k
    q[..., 0], k[..., 0] = 4.0, 0.0
    k[:, 0] = 0.0
    k[:, 0, :, 0] = gap * d ** 0.5 / 4.0
    v = v + 1.0
    v[:, 0] = 0.0
    lengths = torch.tensor([cache - 3], dtype=torch.int32, device=DEV)
    ck = window_kernel(rt, b, new, cache, heads, kv, d, 19000, 2, dtype)
    out = ck(q, k, v, lengths)
    half = half_step(dtype) if ck.kernel.plan.kernels[0].config["kind"] == "tiles" else 2.0 ** -16
    check_attention(out, q, k, v, lengths, 19000, 2, dtype, half)
    assert bool((out > 0).all())


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("use", ["p", "kp", "pm"])
@pytest.mark.parametrize("rows,vocab", [(3, 22670), (18, 164945)])
def test_sample_masks_of_the_lowest_value_in_flat_rows(rt, rows, vocab, use, dtype):
    """Masked tokens that are finite, in rows of which the filters keep too many
    tokens for the packed list."""
    x, u = sample_inputs(rows, vocab, dtype, seed=vocab, spread=1.0)
    g = gen_of(51)
    x[torch.rand(rows, vocab, generator=g, device=DEV) < 0.3] = torch.finfo(x.dtype).min
    params = {"temperature": 1.0 + 7.0 * torch.rand(rows, generator=g, device=DEV)}
    if "k" in use:
        params["top_k"] = torch.full((rows,), vocab * 3 // 5, dtype=torch.int32, device=DEV)
    params["top_p"] = 0.5 + 0.499 * torch.rand(rows, generator=g, device=DEV)
    if "m" in use:
        params["min_p"] = torch.full((rows,), 1e-3, device=DEV)
    ck = compiled(rt, graphs.sample(rows, vocab, dtype=dtype, top_k="k" in use, top_p=True, min_p="m" in use), dtype)
    check_sample(ck(x, u, *params.values()), x, u, **params)


@pytest.mark.parametrize("rows,vocab", [(64, 30011), (24, 131072)])
def test_sample_top_p_next_to_a_running_weight(rt, rows, vocab):
    """top_p within 2e-10 to 1e-9 of what the tokens down to one of them weigh: it
    is the last one kept, or the first one dropped, and u near 1 draws it."""
    x, _ = sample_inputs(rows, vocab, "float32", seed=vocab)
    x = x.sort(-1, descending=True).values
    w = np.exp((x - x[:, :1]).double().cpu().numpy())
    reach = np.cumsum(w, 1) / w.sum(1, keepdims=True)
    p = reach.astype(np.float32)
    off = np.abs(p.astype(np.float64) - reach)
    fits = (reach > 0.6) & (reach < 0.97) & (off > 2e-10) & (off < 1e-9)
    at = fits.argmax(1)
    assert fits.any(1).mean() > 0.9
    top_p = torch.from_numpy(p[np.arange(rows), at]).to(DEV)
    u = torch.full((rows,), 1.0 - 2.0 ** -24, device=DEV)
    t = torch.ones(rows, device=DEV)
    check_sample(compiled(rt, graphs.sample(rows, vocab, top_p=True), "float32")(x, u, t, top_p), x, u, top_p=top_p)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("style", ["half", "interleaved"])
@pytest.mark.parametrize("dim,sections", [(128, [64]), (128, [16, 24, 24]), (6, [1, 1, 1]), (80, [13, 27])])
def test_rope_leaves_padding_as_it_is(rt, dim, sections, style, dtype):
    """Whatever stands in a pair of padding, or past the table, comes out again:
    infinities and NaN, whose partners they must not reach, and -0."""
    b, s, h, rows, axes = 2, 9, 5, 20, len(sections)
    x = torch.randn(b, s, h, dim, generator=gen_of(61), device=DEV)
    odd = torch.tensor([float("inf"), -float("inf"), float("nan"), -0.0, 0.0], device=DEV)
    pick = torch.randint(0, 10, x.shape, generator=gen_of(62), device=DEV)
    x = torch.where(pick < 5, odd[pick.clamp(max=4)], x).to(DT[dtype])
    cos, sin = tables(rows, dim // 2)
    pos = torch.randint(-1, 2, (axes, b, s), generator=gen_of(63), device=DEV, dtype=torch.int32)
    pos[pos == 1] = rows + 3                           # (0: the one that is turned)
    out = compiled(rt, graphs.rope_positions(b, s, h, dim, rows, sections, dtype=dtype, style=style), dtype)(
        x, cos, sin, pos)
    MoltenRuntime.read_status(0)
    axis = torch.repeat_interleave(torch.arange(axes), torch.tensor(sections)).to(DEV)
    stays = (pos[axis] != 0).movedim(0, -1)[:, :, None].expand(b, s, h, dim // 2)      # by pair
    stays = torch.cat((stays, stays), -1) if style == "half" else stays.repeat_interleave(2, -1)
    bits = {2: torch.int16, 4: torch.int32}[x.element_size()]
    same = (out.view(bits) == x.view(bits)) | (torch.isnan(out) & torch.isnan(x))
    assert bool(same[stays].all())
