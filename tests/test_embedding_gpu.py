"""Embedding and its gradient (orda_embedding_device, orda_embedding_grad_device) against 64 bits.

Tolerances (half a step, relative: bf16 2^-8, fp32 2^-24): the forward pass rounds one fp32 product
and, for bf16, that once more. A sum of m rows in fp32 is off by at most (m + 1) 2^-24 times the sum of
their magnitudes, the product with the scale by 2^-24, adding to an old value by 2^-24, and the result's
rounding by half a step of its type.
"""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
STEP = {BF16: 2.0**-8, F32: 2.0**-24}


@pytest.fixture(scope="module")
def ctx():
    from orda_b200.device import DeviceContext

    with DeviceContext(0) as c:
        yield c


def rng(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rand(shape, dtype, gen):
    return torch.randn(*shape, generator=gen, device="cuda").to(dtype)


def skewed(n, v, gen):
    u = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64)
    return torch.exp(u * math.log(v + 1.0)).long().sub_(1).clamp_(0, v - 1)


def finish(ctx):
    torch.cuda.synchronize()
    ctx.check()


@pytest.mark.parametrize("tdt", [BF16, F32])
@pytest.mark.parametrize("odt", [BF16, F32])
@pytest.mark.parametrize("n,h,v", [(1, 1, 1), (1, 8, 5), (3, 7, 100), (33, 64, 1000), (8, 4096, 300), (130, 1001, 50),
                                   (257, 2050, 64), (1000, 100, 2000), (5, 9000, 40)])
def test_forward(ctx, n, h, v, tdt, odt):
    from orda_b200.device import embedding_device

    gen = rng(n + h)
    table, ids = rand((v, h), tdt, gen), torch.randint(0, v, (n,), generator=gen, device="cuda")
    for scale in (1.0, math.sqrt(h)):
        out = embedding_device(ctx, table, ids, scale=scale, dtype=odt)
        finish(ctx)
        want = table.double()[ids] * scale
        assert out.dtype == odt and out.shape == (n, h)
        tol = want.abs() * (2.0**-24 * 2 + STEP[odt]) if scale != 1.0 or tdt != odt else want.abs() * 0
        assert torch.all((out.double() - want).abs() <= tol)


def test_forward_shapes_strides_and_streams(ctx):
    from orda_b200.device import embedding_device

    gen = rng(1)
    base = rand((90, 70), BF16, gen)
    ids = torch.randint(0, 90, (4, 5), generator=gen, device="cuda")
    for table in (base, base[:, 2:66], base[:, 3:66], base[::2][:40, 8:40]):
        idx = ids % table.shape[0]
        out = embedding_device(ctx, table, idx)
        finish(ctx)
        assert out.shape == (4, 5, table.shape[1]) and torch.equal(out, table[idx])
    wide = torch.full((20, 100), 7.0, device="cuda", dtype=BF16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        embedding_device(ctx, base, ids.view(-1), out=wide[:, 8:78])
    torch.cuda.current_stream().wait_stream(side)
    finish(ctx)
    assert torch.equal(wide[:, 8:78], base[ids.view(-1)])
    assert torch.all(wide[:, :8] == 7) and torch.all(wide[:, 78:] == 7)
    empty = embedding_device(ctx, base, torch.empty(0, dtype=torch.int64, device="cuda"))
    assert empty.shape == (0, 70)


def grad_formula(g, ids, v, scale, old=None, padding=None):
    """The gradient and its bound but for the output's rounding, in 64 bits."""
    h = g.shape[1]
    keep = torch.ones_like(ids, dtype=torch.bool) if padding is None else ids != padding
    s = torch.zeros(v, h, dtype=torch.float64, device="cuda").index_add_(0, ids[keep], g.double()[keep])
    mag = torch.zeros(v, h, dtype=torch.float64, device="cuda").index_add_(0, ids[keep], g.double()[keep].abs())
    m = torch.bincount(ids[keep], minlength=v)[:, None]
    want = s * scale
    tol = mag * abs(scale) * 2.0**-24 * (m + 2)
    if old is not None:
        want = want + old.double()
        tol = tol + 2.0**-24 * want.abs()
    return want, tol


def check_grad(got, want, tol):
    step = STEP[got.dtype]
    off = (got.double() - want).abs() - (tol + step * (want.abs() + tol))
    assert off.max() <= 0, float(off.max())


SIZES = [(1, 1, 1), (1, 64, 10), (2, 9, 3), (7, 100, 1), (8, 8, 512), (9, 64, 511), (40, 1001, 17), (257, 128, 70000),
         (1000, 33, 5), (2047, 2050, 300), (2048, 72, 513), (8191, 256, 2000), (9000, 40, 300000), (40000, 16, 40)]


@pytest.mark.parametrize("gdt,odt", [(BF16, BF16), (BF16, F32), (F32, F32), (F32, BF16)])
@pytest.mark.parametrize("n,h,v", SIZES)
def test_gradient(ctx, n, h, v, gdt, odt):
    from orda_b200.device import embedding_grad_device

    gen = rng(n + v)
    g, ids = rand((n, h), gdt, gen), skewed(n, v, gen)
    scale = math.sqrt(h)
    got = embedding_grad_device(ctx, g, ids, v, scale=scale, dtype=odt)
    finish(ctx)
    assert got.shape == (v, h) and got.dtype == odt
    want, tol = grad_formula(g, ids, v, scale)
    check_grad(got, want, tol)
    assert not got[torch.bincount(ids, minlength=v) == 0].any()
    # on top of a gradient, twice; rows that no token names keep their bits
    acc = rand((v, h), odt, gen)
    for _ in range(2):
        old = acc.clone()
        embedding_grad_device(ctx, g, ids, v, scale=scale, out=acc, accumulate=True)
        finish(ctx)
        check_grad(acc, *grad_formula(g, ids, v, scale, old=old))
        untouched = torch.bincount(ids, minlength=v) == 0
        assert torch.equal(acc[untouched], old[untouched])


@pytest.mark.parametrize("n,v", [(5000, 300), (12345, 131072), (64, 8)])
def test_orders_and_runs(ctx, n, v):
    """Ids that are all the same, sorted, reversed, and one run over most tiles between short ones."""
    from orda_b200.device import embedding_grad_device

    gen = rng(n)
    h = 136
    g = rand((n, h), BF16, gen)
    one = torch.full((n,), v - 1, device="cuda")
    up = torch.sort(torch.randint(0, v, (n,), generator=gen, device="cuda")).values
    mixed = torch.randint(0, v, (n,), generator=gen, device="cuda")
    mixed[n // 10: -(n // 10)] = v // 2
    for ids in (one, up, up.flip(0), mixed, torch.arange(n, device="cuda") % v):
        ids = ids.contiguous()
        got = embedding_grad_device(ctx, g, ids, v, dtype=F32)
        again = embedding_grad_device(ctx, g, ids, v, dtype=F32)
        finish(ctx)
        check_grad(got, *grad_formula(g, ids, v, 1.0))
        assert torch.equal(got, again)


def test_padding_id(ctx):
    from orda_b200.device import embedding_grad_device

    gen = rng(3)
    n, h, v = 3000, 64, 50
    g, ids = rand((n, h), BF16, gen), skewed(n, v, gen)
    for pad in (0, 7, 49):
        got = embedding_grad_device(ctx, g, ids, v, padding_id=pad, dtype=F32)
        finish(ctx)
        assert not got[pad].any()
        check_grad(got, *grad_formula(g, ids, v, 1.0, padding=pad))
        # what a padding token's row holds is not used
        g2 = g.clone()
        g2[ids == pad] = float("nan")
        assert torch.equal(got, embedding_grad_device(ctx, g2, ids, v, padding_id=pad, dtype=F32))
    # a padding id outside the table names nothing, and is no bad id
    ids[::5] = -1
    got = embedding_grad_device(ctx, g, ids, v, padding_id=-1, dtype=F32)
    finish(ctx)
    check_grad(got, *grad_formula(g[ids >= 0], ids[ids >= 0], v, 1.0))
    assert not embedding_grad_device(ctx, g, torch.full_like(ids, 4), v, padding_id=4).any()


def test_gradient_strides_and_no_tokens(ctx):
    from orda_b200.device import embedding_grad_device

    gen = rng(4)
    n, v = 500, 120
    ids = skewed(n, v, gen)
    base = rand((n, 200), BF16, gen)
    for lo, hi in ((0, 200), (8, 136), (3, 64)):
        g = base[:, lo:hi]
        full = torch.full((v, 211), 7.0, device="cuda")
        out = full[:, 5:5 + hi - lo]
        embedding_grad_device(ctx, g, ids, v, out=out)
        finish(ctx)
        check_grad(out, *grad_formula(g, ids, v, 1.0))
        assert torch.all(full[:, :5] == 7) and torch.all(full[:, 5 + hi - lo:] == 7)
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    got = embedding_grad_device(ctx, base[:0], none, v)
    finish(ctx)
    assert got.shape == (v, 200) and not got.any()
    keep = rand((v, 200), BF16, gen)
    assert torch.equal(embedding_grad_device(ctx, base[:0], none, v, out=keep.clone(), accumulate=True), keep)


def test_bad_ids_are_reported_and_do_nothing(ctx):
    import orda_b200 as ob
    from orda_b200 import _abi
    from orda_b200.device import embedding_device, embedding_grad_device, linear_cross_entropy_device

    gen = rng(5)
    n, h, v = 100, 64, 40
    ids = skewed(n, v, gen)
    bad = ids.clone()
    bad[3], bad[50], bad[99] = -1, v, 2**40
    good = (bad >= 0) & (bad < v)
    table, g = rand((v, h), BF16, gen), rand((n, h), BF16, gen)
    out = embedding_device(ctx, table, bad)
    # the report outlives calls in between
    linear_cross_entropy_device(ctx, g, table, ids)
    with pytest.raises(ob.OrdaError, match="token id") as e:
        ctx.check()
    assert e.value.code == _abi.ORDA_ERR_LABEL
    assert torch.equal(out[good], table[bad[good]]) and not out[~good].any()
    ctx.check()
    got = embedding_grad_device(ctx, g, bad, v, dtype=F32)
    with pytest.raises(ob.OrdaError, match="token id"):
        ctx.check()
    check_grad(got, *grad_formula(g[good], bad[good], v, 1.0))
    ctx.check()


def test_refusals(ctx):
    import orda_b200 as ob
    from orda_b200.device import embedding_device, embedding_grad_device

    table = torch.zeros(10, 8, device="cuda", dtype=BF16)
    ids = torch.zeros(4, device="cuda", dtype=torch.int64)
    g = torch.zeros(4, 8, device="cuda", dtype=BF16)
    with pytest.raises(ValueError, match="dtype"):
        embedding_device(ctx, table.half(), ids)
    with pytest.raises(ob.OrdaError, match="finite"):
        embedding_device(ctx, table, ids, scale=float("inf"))
    with pytest.raises(ValueError, match="rows of"):
        embedding_device(ctx, table, ids, out=torch.zeros(3, 8, device="cuda"))
    with pytest.raises(ob.OrdaError, match="2\\^20"):
        embedding_device(ctx, torch.zeros(1, 2**20 + 8, device="cuda", dtype=BF16), ids)
    with pytest.raises(ob.OrdaError, match="ld >= H"):
        embedding_grad_device(ctx, g, ids, 10, out=torch.zeros(1, 8, device="cuda").expand(10, 8))
    with pytest.raises(ValueError, match="accumulate"):
        embedding_grad_device(ctx, g, ids, 10, accumulate=True)
    with pytest.raises(ValueError, match="rows of"):
        embedding_grad_device(ctx, g[:3], ids, 10)
    with pytest.raises(ValueError, match=r"\(10, 8\)"):
        embedding_grad_device(ctx, g, ids, 10, out=torch.zeros(10, 9, device="cuda"))
    finish(ctx)


def test_gradient_against_differences(ctx):
    """The gradient of sum(c * embedding) by differences in 64 bits: it is linear in the table."""
    from orda_b200.device import embedding_device, embedding_grad_device

    gen = rng(6)
    n, h, v = 60, 24, 11
    ids, c = skewed(n, v, gen), rand((n, h), F32, gen)
    d = rand((v, h), F32, gen)
    got = embedding_grad_device(ctx, c, ids, v, scale=3.0)
    f = lambda t: float((embedding_device(ctx, t, ids, scale=3.0).double() * c.double()).sum())  # noqa: E731
    t0 = rand((v, h), F32, gen)
    want = (f(t0 + d) - f(t0 - d)) / 2
    finish(ctx)
    # every product and sum of f is off by 2^-24 of its magnitude at most, three roundings each
    mag = float((3.0 * ((t0.abs() + d.abs())[ids] * c.abs())).sum())
    assert abs(float((got.double() * d.double()).sum()) - want) <= 4 * 2.0**-24 * mag * (n + 3)


def test_captured(ctx):
    from orda_b200.device import DeviceContext, embedding_device, embedding_grad_device

    gen = rng(7)
    n, h, v = 600, 64, 900
    table, g = rand((v, h), BF16, gen), rand((n, h), BF16, gen)
    ids = skewed(n, v, gen)
    with DeviceContext(0) as own:
        embedding_grad_device(own, g, ids, v)
        x, dt = torch.empty(n, h, device="cuda", dtype=BF16), torch.empty(v, h, device="cuda", dtype=BF16)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            embedding_device(own, table, ids, out=x)
            embedding_grad_device(own, g, ids, v, out=dt)
        embedding_grad_device(own, rand((20000, h), BF16, gen), skewed(20000, v, gen), v)  # outgrows the workspace
        for _ in range(2):
            ids.copy_(skewed(n, v, gen))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(x, table[ids])
            assert torch.equal(dt, embedding_grad_device(own, g, ids, v))
        finish(own)
        del graph


def test_shared_table_step(ctx):
    """Embedding, the loss at the output head and both gradients of the one table, as in a training step."""
    from orda_b200.device import embedding_device, embedding_grad_device, linear_cross_entropy_device

    gen = rng(8)
    n, h, v = 300, 128, 1000
    table = (torch.randn(v, h, generator=gen, device="cuda") * 0.1).to(BF16)
    ids = skewed(n, v, gen)
    labels = torch.roll(ids, -1)
    labels[-1] = -100
    scale = math.sqrt(h)
    x = embedding_device(ctx, table, ids, scale=scale)
    r = linear_cross_entropy_device(ctx, x, table, labels)
    head = r.grad_weight.clone()
    embedding_grad_device(ctx, r.grad_hidden, ids, v, scale=scale, out=r.grad_weight, accumulate=True)
    finish(ctx)
    check_grad(r.grad_weight, *grad_formula(r.grad_hidden, ids, v, scale, old=head))
    t = table.double().requires_grad_()
    z = (t[ids] * scale) @ t.T
    loss = torch.nn.functional.cross_entropy(z, labels)
    loss.backward()
    # x is rounded to bf16 (2^-8 of it, once) and so are the logit gradients: three such roundings, rms 1.6e-3 each
    assert abs(loss.item() - float(r.loss)) <= 2.0**-8 * float(z.detach().abs().max())
    assert ((r.grad_weight.double() - t.grad).norm() / t.grad.norm()) < 3 * 2.0**-8


@pytest.mark.parametrize("n", [1, 2, 255, 256, 257, 511, 512, 513, 600, 1023, 1024, 1025])
def test_few_tokens_and_the_sorted_path(ctx, n):
    """Around the token count where the sort takes over; runs over several lookups of 256 ids."""
    from orda_b200.device import embedding_grad_device

    gen = rng(n)
    for h, v in ((40, 3), (2056, 900)):
        g = rand((n, h), BF16, gen)
        for ids in (skewed(n, v, gen), torch.full((n,), v - 1, device="cuda"), torch.arange(n, device="cuda") % v):
            got = embedding_grad_device(ctx, g, ids, v, scale=0.5, dtype=F32)
            finish(ctx)
            check_grad(got, *grad_formula(g, ids, v, 0.5))


def test_offsets_beyond_32_bits(ctx):
    """A table of 2.4e9 elements."""
    from orda_b200.device import embedding_device, embedding_grad_device

    gen = rng(9)
    v, h = 590000, 4096
    table = torch.zeros(v, h, device="cuda", dtype=BF16)
    for n in (40, 700):
        ids = torch.randint(v - 5000, v, (n,), generator=gen, device="cuda")
        ids[::3] = torch.randint(0, 50, (len(ids[::3]),), generator=gen, device="cuda")
        rows = rand((n, h), BF16, gen)
        table[ids] = rows
        assert torch.equal(embedding_device(ctx, table, ids), table[ids])
        got = embedding_grad_device(ctx, rows, ids, v)
        finish(ctx)
        named, back = torch.unique(ids, return_inverse=True)
        check_grad(got[named], *grad_formula(rows, back, len(named), 1.0))
        got[named] = 0
        assert not got.any()
        del got


def test_two_contexts_at_once(ctx):
    from orda_b200.device import DeviceContext, embedding_grad_device

    gen = rng(10)
    with DeviceContext(0) as a, DeviceContext(0) as b:
        work = []
        for c, n, v in ((a, 9000, 4000), (b, 5000, 70000)):
            g, ids = rand((n, 512), BF16, gen), skewed(n, v, gen)
            work.append((c, g, ids, v, embedding_grad_device(c, g, ids, v)))
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        outs = [[], []]
        for _ in range(5):
            for k, (c, g, ids, v, _) in enumerate(work):
                with torch.cuda.stream(streams[k]):
                    outs[k].append(embedding_grad_device(c, g, ids, v))
        torch.cuda.synchronize()
        for k in range(2):
            assert all(torch.equal(o, work[k][4]) for o in outs[k])

@pytest.mark.parametrize("n", [1500, 20000])
@pytest.mark.parametrize("v", [1, 2, 3, 7, 20])
def test_sort_of_few_different_ids(ctx, n, v):
    """Fewer digits than a warp has lanes in the sort."""
    from orda_b200.device import embedding_grad_device

    gen = rng(n + v)
    for h in (24, 2056):
        g, ids = rand((n, h), BF16, gen), torch.randint(0, v, (n,), generator=gen, device="cuda")
        got = embedding_grad_device(ctx, g, ids, v, dtype=F32)
        acc = got.clone()
        embedding_grad_device(ctx, g, ids, v, out=acc, accumulate=True)
        finish(ctx)
        check_grad(got, *grad_formula(g, ids, v, 1.0))
        check_grad(acc, *grad_formula(g, ids, v, 1.0, old=got))
