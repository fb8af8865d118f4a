"""Linear cross entropy (orda_linear_cross_entropy_device) against its formula in 64 bits.

Tolerances, from the arithmetic (u = half a step, relative: bf16 2^-8, fp32 2^-24):
  logits    fp32 sums of H exact products: |dz| <= 2 H 2^-24 sum_k |h_k w_k| (twice the bound of a
            rounded sum, for an accumulator that cuts instead of rounding); nll and lse move by at most
            the largest two such errors, plus 2^-20 for the exponentials and the rounding of the result
  dlogits   2^-8 |dz| for the rounding to bf16, 2^-10 ln 2 p g for the fixed-point logits, and the
            logits' own error and 2^-18 (exponentials of arguments up to 64) in p g
  gradients the sum of the dlogits' errors times |W| (or |h|), K 2^-23 for the fp32 sums, and half a
            step of the output's type
"""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

LN2 = math.log(2.0)


@pytest.fixture(scope="module")
def ctx():
    from orda_b200.device import DeviceContext

    with DeviceContext(0) as c:
        yield c


def make(bt, h, v, seed=0, ignored=0.0, std=0.5, ld=None, pull=0.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    ld = ld or -(-h // 8) * 8
    w = torch.zeros(v, ld, device="cuda", dtype=torch.bfloat16)[:, :h]
    w.copy_(torch.randn(v, h, generator=gen, device="cuda") * (std / math.sqrt(h)))
    labels = torch.randint(0, v, (bt,), generator=gen, device="cuda")
    x = torch.zeros(bt, ld, device="cuda", dtype=torch.bfloat16)[:, :h]
    x.copy_(torch.randn(bt, h, generator=gen, device="cuda") * 2.0 + pull * w[labels].float() * h)
    if ignored:
        labels[torch.rand(bt, generator=gen, device="cuda") < ignored] = -100
    return x, w, labels


def formula(x, w, labels, a=0.0, mean=True, denom=None, ignore=-100):
    """loss, nll, lse, dh, dW and the error bounds of the last four, in 64 bits."""
    live = labels != ignore
    xd = torch.where(live[:, None], x.double(), 0.0)
    wd = w.double()
    v, h = wd.shape
    z = xd @ wd.T
    lse = torch.logsumexp(z, 1)
    y = torch.where(live, labels, 0)
    zy = z.gather(1, y[:, None])[:, 0]
    nll = torch.where(live, lse - (1 - a) * zy - a * z.mean(1), 0.0)
    n = denom or max(int(live.sum()), 1)
    g = torch.where(live, 1.0 / n if mean else 1.0, 0.0)
    p = torch.exp(z - lse[:, None])
    dz = p - a / v
    # the label's entry through 1 - p = the sum of the others: p itself may round to 1 in 64 bits
    miss = p.scatter(1, y[:, None], 0.0).sum(1)
    dz[torch.arange(len(y), device="cuda"), y] = a - a / v - miss
    dz = dz * g[:, None]
    dh, dw = dz @ wd, dz.T @ xd
    ez = 2 * h * 2.0**-24 * (xd.abs() @ wd.abs().T).amax(1)
    row_tol = 2 * ez + 2.0**-20 * (1 + lse.abs() + zy.abs() + z.abs().amax(1))
    pg = p * g[:, None]
    err = 2.0**-8 * dz.abs() + pg * (2.0**-10 * LN2 + 2.0**-18 + 3 * ez[:, None])
    # the label's entry is formed from 1 - p
    mag = dz.abs() + pg
    dh_tol = err @ wd.abs() + 2.0**-23 * v * (mag @ wd.abs()) / max(1.0, math.sqrt(v))
    dw_tol = err.T @ xd.abs() + 2.0**-23 * len(y) * (mag.T @ xd.abs())
    return {"loss": nll.sum() / n if mean else nll.sum(), "nll": nll, "lse": torch.where(live, lse, 0.0), "dh": dh,
            "dw": dw, "row_tol": row_tol, "dh_tol": dh_tol, "dw_tol": dw_tol, "dz": dz, "n": n}


def check(r, f, mean=True):
    assert torch.all((r.nll.double() - f["nll"]).abs() <= f["row_tol"] + 2.0**-23 * f["nll"].abs()), "nll"
    assert torch.all((r.lse.double() - f["lse"]).abs() <= f["row_tol"] + 2.0**-23 * f["lse"].abs()), "lse"
    tol = f["row_tol"].sum() / (f["n"] if mean else 1) + 2.0**-22 * f["loss"].abs()
    assert (r.loss.double() - f["loss"]).abs() <= tol, (float(r.loss), float(f["loss"]))
    for got, want, tol in ((r.grad_hidden, f["dh"], f["dh_tol"]), (r.grad_weight, f["dw"], f["dw_tol"])):
        if got is None:
            continue
        step = 2.0**-8 if got.dtype == torch.bfloat16 else 2.0**-24
        off = (got.double() - want).abs() - (tol + step * (want.abs() + tol) + 1e-38)
        assert off.max() <= 0, (float(off.max()), float(want.abs().max()))


def call(ctx, x, w, labels, a=0.0, mean=True, **kw):
    import orda_b200 as ob
    from orda_b200.device import linear_cross_entropy_device

    r = linear_cross_entropy_device(ctx, x, w, labels, label_smoothing=a,
                                    reduction=ob.Reduction.Mean if mean else ob.Reduction.Sum, **kw)
    torch.cuda.synchronize()
    ctx.check()
    return r


SHAPES = [(1, 8, 1), (1, 8, 2), (3, 16, 5), (1, 64, 1000), (2, 72, 127), (31, 64, 128), (33, 136, 129), (127, 128, 255),
          (128, 256, 257), (129, 8, 513), (257, 1000, 1031), (300, 520, 4099), (640, 264, 2500)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bt,h,v", SHAPES)
def test_shapes(ctx, bt, h, v, dtype):
    x, w, labels = make(bt, h, v, seed=bt + v)
    check(call(ctx, x, w, labels, grad_dtype=dtype), formula(x, w, labels))


@pytest.mark.parametrize("bt,h,v", [(33, 136, 129), (300, 520, 4099)])
@pytest.mark.parametrize("a,mean,ignored", [(0.1, True, 0.0), (1.0, True, 0.3), (0.1, False, 0.5), (0.0, False, 0.9)])
def test_options(ctx, bt, h, v, a, mean, ignored):
    x, w, labels = make(bt, h, v, seed=7, ignored=ignored)
    r = call(ctx, x, w, labels, a, mean, grad_dtype=torch.bfloat16)
    check(r, formula(x, w, labels, a, mean), mean)
    dead = labels == -100
    assert torch.all(r.nll[dead] == 0) and torch.all(r.lse[dead] == 0) and torch.all(r.grad_hidden[dead] == 0)


@pytest.mark.parametrize("piece_bytes", [1, 300 * 1024 * 2, 300 * 1600 * 2])
@pytest.mark.parametrize("a", [0.0, 0.2])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_pieces(ctx, piece_bytes, a, dtype):
    """The vocabulary in 9, 5 and 3 pieces (the last one narrow)."""
    x, w, labels = make(300, 264, 4099, seed=3, ignored=0.2)
    check(call(ctx, x, w, labels, a, grad_dtype=dtype, piece_bytes=piece_bytes), formula(x, w, labels, a))


def test_odd_h_and_row_strides(ctx):
    x, w, labels = make(70, 61, 333, seed=5, ld=72)
    assert x.stride(0) == 72
    check(call(ctx, x, w, labels, grad_dtype=torch.bfloat16), formula(x, w, labels))
    # outputs that no TMA store can address
    for dtype in (torch.bfloat16, torch.float32):
        out = {"grad_hidden": torch.full((70, 67), 7.0, device="cuda", dtype=dtype)[:, 3:64],
               "grad_weight": torch.full((333, 67), 7.0, device="cuda", dtype=dtype)[:, 3:64]}
        full = {k: t._base for k, t in out.items()}
        r = call(ctx, x, w, labels, out=out)
        check(r, formula(x, w, labels))
        for t in full.values():
            assert torch.all(t[:, :3] == 7.0) and torch.all(t[:, 64:] == 7.0)


@pytest.mark.parametrize("need_h,need_w", [(False, False), (True, False), (False, True)])
def test_gradients_asked_for(ctx, need_h, need_w):
    x, w, labels = make(130, 128, 1500, seed=9, ignored=0.1)
    f = formula(x, w, labels)
    for pieces in (0, 1):
        r = call(ctx, x, w, labels, need_grad_hidden=need_h, need_grad_weight=need_w, piece_bytes=pieces)
        assert (r.grad_hidden is not None) == need_h and (r.grad_weight is not None) == need_w
        check(r, f)


@pytest.mark.parametrize("piece_bytes", [0, 1])
def test_far_labels(ctx, piece_bytes):
    """Labels whose logit lies far below or above every other one: parts outside the fixed point's range."""
    bt, h, v = 96, 64, 1200
    gen = torch.Generator(device="cuda").manual_seed(2)
    w = torch.zeros(v, h, device="cuda")
    w[:, 0] = torch.linspace(-1, 1, v, device="cuda")
    w[:, 1:] = torch.randn(v, h - 1, generator=gen, device="cuda") * 0.1
    w = w.bfloat16()
    x = torch.randn(bt, h, generator=gen, device="cuda")
    x[:, 0] = torch.linspace(-150, 150, bt, device="cuda")  # logits up to +-150 (e^300 apart)
    x = x.bfloat16()
    labels = torch.randint(0, v, (bt,), generator=gen, device="cuda")
    labels[::3] = 0
    labels[1::3] = v - 1
    r = call(ctx, x, w, labels, grad_dtype=torch.bfloat16, piece_bytes=piece_bytes)
    check(r, formula(x, w, labels))
    # rows that are all but certain: the gradient's scale is 1 - p, far below a rounding of p
    sure = torch.zeros(4, h, device="cuda", dtype=torch.bfloat16)
    sure[:, 0] = 40.0
    lab = torch.full((4,), v - 1, device="cuda")
    w2 = w.clone()
    w2[:-1, 0] = -1.0
    f = formula(sure, w2, lab)
    r = call(ctx, sure, w2, lab, piece_bytes=piece_bytes)
    rel = ((r.grad_hidden.double() - f["dh"]).norm() / f["dh"].norm()).item()
    assert float(f["dh"].norm()) < 1e-25 and rel < 1e-2, rel
    assert torch.allclose(r.nll.double(), f["nll"], rtol=1e-3, atol=0) or float(f["nll"].max()) < 1e-12


def test_nothing_of_an_ignored_row_is_used(ctx):
    x, w, labels = make(140, 96, 700, seed=4, ignored=0.4)
    dead = labels == -100
    clean = call(ctx, x, w, labels)
    for bad in (float("nan"), float("inf"), -torch.finfo(torch.bfloat16).max):
        y = x.clone()
        y[dead] = bad
        r = call(ctx, y, w, labels)
        for n in ("loss", "nll", "lse", "grad_hidden", "grad_weight"):
            assert torch.equal(getattr(r, n), getattr(clean, n)), (bad, n)


def test_every_row_ignored(ctx):
    x, w, labels = make(65, 64, 300)
    labels.fill_(-100)
    for a, mean in ((0.0, True), (0.1, False)):
        r = call(ctx, x, w, labels, a, mean)
        assert float(r.loss) == 0 and not r.grad_hidden.any() and not r.grad_weight.any() and not r.lse.any()


def test_nan_of_a_live_row_shows(ctx):
    x, w, labels = make(40, 64, 300)
    x[3, 5] = float("nan")
    r = call(ctx, x, w, labels)
    assert torch.isnan(r.loss) and torch.isnan(r.nll[3]) and torch.isnan(r.grad_hidden[3]).all()
    assert torch.isfinite(r.nll[[i for i in range(40) if i != 3]]).all()


def test_lowest_value_logits(ctx):
    """Vocabulary entries that are masked by a large negative logit."""
    x, w, labels = make(64, 64, 640, seed=6)
    x[:, 0] = 1.0
    w[:, 0] = 0.0
    w[128:384, 0] = -3.0e38
    labels[(labels >= 128) & (labels < 384)] = 5
    r = call(ctx, x, w, labels, grad_dtype=torch.bfloat16)
    keep = torch.cat([torch.arange(128), torch.arange(384, 640)]).cuda()
    sub = torch.full((640,), 0, device="cuda")
    sub[keep] = torch.arange(len(keep), device="cuda")
    f = formula(x, w[keep].contiguous(), sub[labels])
    assert torch.all((r.nll.double() - f["nll"]).abs() <= f["row_tol"])
    assert not r.grad_weight[128:384].any()
    assert ((r.grad_weight[keep].double() - f["dw"]).norm() / f["dw"].norm()) < 5e-3


def test_label_out_of_range_is_reported(ctx):
    import orda_b200 as ob
    from orda_b200 import _abi
    from orda_b200.device import linear_cross_entropy_device

    x, w, labels = make(40, 64, 300)
    for bad in (300, -1):
        labels[7] = bad
        linear_cross_entropy_device(ctx, x, w, labels)
        with pytest.raises(ob.OrdaError) as e:
            ctx.check()
        assert e.value.code == _abi.ORDA_ERR_LABEL
    labels[7] = 2
    check(call(ctx, x, w, labels), formula(x, w, labels))


def test_own_ignore_index_and_denominator(ctx):
    x, w, labels = make(90, 64, 300, seed=8)
    labels[::4] = 17
    r = call(ctx, x, w, labels, ignore_index=17)
    check(r, formula(x, w, labels, ignore=17))
    r = call(ctx, x, w, labels, global_non_ignore=1000)
    check(r, formula(x, w, labels, denom=1000))


def test_gradient_against_differences(ctx):
    """Directional derivatives of the 64-bit loss by central differences."""
    x, w, labels = make(50, 72, 401, seed=12, ignored=0.2)
    r = call(ctx, x, w, labels, 0.1)
    gen = torch.Generator(device="cuda").manual_seed(1)
    for i in range(4):
        dx = torch.randn(x.shape, generator=gen, device="cuda", dtype=torch.float64)
        dw = torch.randn(w.shape, generator=gen, device="cuda", dtype=torch.float64) / 72
        eps = 1e-4
        up = formula(x.double() + eps * dx, w.double() + eps * dw, labels, 0.1)["loss"]
        down = formula(x.double() - eps * dx, w.double() - eps * dw, labels, 0.1)["loss"]
        f = formula(x, w, labels, 0.1)
        want = float((up - down) / (2 * eps))
        got = float((r.grad_hidden.double() * dx).sum() + (r.grad_weight.double() * dw).sum())
        tol = float((f["dh_tol"] * dx.abs()).sum() + (f["dw_tol"] * dw.abs()).sum()) + 1e-6
        assert abs(got - want) <= tol, (got, want, tol)


def test_same_bits_twice_and_on_another_stream(ctx):
    x, w, labels = make(520, 200, 9000, seed=10, ignored=0.1)
    for piece in (0, 520 * 2048 * 2):
        a = call(ctx, x, w, labels, piece_bytes=piece)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            b = call(ctx, x, w, labels, piece_bytes=piece)
        torch.cuda.current_stream().wait_stream(side)
        for n in ("loss", "nll", "lse", "grad_hidden", "grad_weight"):
            assert torch.equal(getattr(a, n), getattr(b, n)), n


def test_captured_call_replays_after_the_workspace_grew(ctx):
    from orda_b200.device import DeviceContext, linear_cross_entropy_device

    x, w, labels = make(100, 128, 2000, seed=11)
    with DeviceContext(0) as own:
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(Exception, match="before the capture"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                linear_cross_entropy_device(own, x, w, labels)
        torch.cuda.synchronize()
        call(own, x, w, labels)
        out = {"loss": torch.zeros(1, device="cuda"), "grad_hidden": torch.zeros(100, 128, device="cuda"),
               "grad_weight": torch.zeros(2000, 128, device="cuda")}
        with torch.cuda.graph(graph):
            linear_cross_entropy_device(own, x, w, labels, out=out)
        big = make(400, 256, 5000, seed=13)
        call(own, *big)
        for seed in (21, 22):
            x2, w2, l2 = make(100, 128, 2000, seed=seed, ignored=0.3)
            x.copy_(x2), w.copy_(w2), labels.copy_(l2)
            graph.replay()
            torch.cuda.synchronize()
            eager = call(own, x, w, labels)
            assert torch.equal(eager.grad_weight, out["grad_weight"])
            assert torch.equal(eager.grad_hidden, out["grad_hidden"]) and float(out["loss"]) == float(eager.loss)
        del graph


def test_allocation_failures_make_smaller_pieces(ctx):
    from orda_b200.device import DeviceContext

    x, w, labels = make(64, 64, 3000, seed=14)
    with DeviceContext(0) as own:
        own.inject_alloc_failures(2)
        check(call(own, x, w, labels), formula(x, w, labels))
        own.inject_alloc_failures(100)
        with pytest.raises(RuntimeError, match="workspace"):
            call(own, x, w, labels)
        own.inject_alloc_failures(0)


def test_agrees_with_the_distillation_losss_student_term(ctx):
    """kd = 0 and no teacher CE leave the distillation loss its student term."""
    import orda_b200 as ob
    from orda_b200.device import distillation_loss_device

    x, w, labels = make(200, 128, 1500, seed=15, ignored=0.2)
    d = distillation_loss_device(ctx, x, w, labels, ob.TeacherMode.Tied, teacher_hidden=x,
                                 opts=ob.LossOptions(kd_weight=0.0, teacher_ce_weight=0.0, label_smoothing=0.1))
    torch.cuda.synchronize()
    r = call(ctx, x, w, labels, 0.1)
    f = formula(x, w, labels, 0.1)
    tol = float(f["row_tol"].max())
    assert abs(float(d.scalars[1]) - float(r.loss)) <= 2 * tol
    for a, b, t in ((d.grad_student_hidden, r.grad_hidden, f["dh_tol"]), (d.grad_weight, r.grad_weight, f["dw_tol"])):
        assert torch.all((a.double() - b.double()).abs() <= 2 * t + 1e-30)


@pytest.mark.parametrize("pull", [0.5, 0.05])
@pytest.mark.parametrize("bt,h,v", [(2048, 1024, 12000), (700, 2048, 20011)])
def test_larger_products(ctx, bt, h, v, pull):
    """Full tiles, wide tiles and slabs; relative L2 of three bf16 roundings (1.6e-3 rms each) at most.
    pull = 0.05 lifts the labels' logits by about 13 (H = 1024), 0.5 by 128: there the gradients are
    about e^-128 = 2.6e-56, below what bf16 and fp32 hold, so an element may be off by 2^-126, where the
    arithmetic flushes to zero."""
    x, w, labels = make(bt, h, v, seed=16, pull=pull, ignored=0.1)
    for piece in (0, bt * v // 2):
        r = call(ctx, x, w, labels, grad_dtype=torch.bfloat16, piece_bytes=piece)
        f = formula(x, w, labels)
        check(r, f)
        for got, want in ((r.grad_hidden, f["dh"]), (r.grad_weight, f["dw"])):
            flushed = math.sqrt(want.numel()) * 2.0**-126
            assert (got.double() - want).norm() < 1.6e-3 * math.sqrt(3) * want.norm() + flushed


@pytest.mark.parametrize("bt", [1, 31, 32, 33, 64, 65, 127, 128, 129])
@pytest.mark.parametrize("a", [0.0, 0.1])
def test_few_rows(ctx, bt, a):
    """Around the row counts at which the logits' kernel changes, whole and in pieces."""
    x, w, labels = make(bt, 200, 2531, seed=bt, ignored=0.2 if bt > 4 else 0.0)
    f = formula(x, w, labels, a)
    for piece in (0, bt * 1024 * 2):
        check(call(ctx, x, w, labels, a, grad_dtype=torch.bfloat16, piece_bytes=piece), f)
    check(call(ctx, x, w, labels, a, need_grad_hidden=False, need_grad_weight=False), f)


def test_refusals(ctx):
    import orda_b200 as ob
    from orda_b200.device import linear_cross_entropy_device as f

    x, w, labels = make(20, 64, 100)
    for args, kw, what in [
        ((x, w, labels), {"label_smoothing": 1.5}, "label_smoothing"),
        ((x, w, labels), {"label_smoothing": float("nan")}, "label_smoothing"),
        ((x, w, labels), {"reduction": 7}, "reduction"),
        ((x, w, labels), {"global_non_ignore": -1}, "global_non_ignore"),
        ((x, w, labels[:19].clone()), {}, "BT=20"),
        ((x, w[:, :56], labels), {}, "weight must be"),
        ((x[:0], w, labels[:0]), {}, "BT must be > 0"),
        ((x.float(), w, labels), {}, "bf16"),
        ((x, w[:, 1:57], labels), {}, "weight must be"),
        ((x[:, 1:57], w[:, 1:57], labels), {}, "16-byte aligned"),
        ((x[:1].expand(20, 64), w, labels), {}, "16-byte aligned"),
        ((x, w, labels), {"out": {"grad_weight": torch.zeros(1, 64, device="cuda").expand(100, 64)}}, "ld >= H"),
    ]:
        with pytest.raises(ob.OrdaError, match=what):
            f(ctx, *args, **kw)
    for kw, what in [({"out": {"loss": torch.zeros(2, device="cuda")}}, "loss"),
                     ({"out": {"nll": torch.zeros(20, device="cuda", dtype=torch.float64)}}, "nll"),
                     ({"out": {"grad_hidden": torch.zeros(20, 65, device="cuda")}}, "grad_hidden"),
                     ({"out": {"grad_hidden": torch.zeros(20, 64, device="cuda")}, "need_grad_hidden": False}, "need_"),
                     ({"grad_dtype": torch.float16}, "dtype")]:
        with pytest.raises(ValueError, match=what):
            f(ctx, x, w, labels, **kw)
    check(call(ctx, x, w, labels), formula(x, w, labels))


def test_two_graphs_share_a_context(ctx):
    from orda_b200.device import DeviceContext, linear_cross_entropy_device

    cases = [make(100, 128, 2000, seed=31), make(300, 64, 5000, seed=32, ignored=0.3)]
    with DeviceContext(0) as own:
        want = [call(own, *c) for c in cases]
        graphs, outs = [], []
        for c in cases:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                outs.append(linear_cross_entropy_device(own, *c))
            graphs.append(g)
        for _ in range(3):
            for g in graphs:
                g.replay()
        torch.cuda.synchronize()
        for r, f in zip(outs, want):
            for n in ("loss", "nll", "lse", "grad_hidden", "grad_weight"):
                assert torch.equal(getattr(r, n), getattr(f, n)), n
        del graphs


def test_two_contexts_at_once(ctx):
    from orda_b200.device import DeviceContext, linear_cross_entropy_device

    cases = [make(200, 128, 9000, seed=41), make(40, 512, 20000, seed=42)]
    with DeviceContext(0) as a, DeviceContext(0) as b:
        want = [call(c, *case) for c, case in zip((a, b), cases)]
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        got = [[], []]
        for _ in range(5):
            for k, c in enumerate((a, b)):
                with torch.cuda.stream(streams[k]):
                    got[k].append(linear_cross_entropy_device(c, *cases[k]))
        torch.cuda.synchronize()
        for k in range(2):
            for r in got[k]:
                assert torch.equal(r.grad_weight, want[k].grad_weight) and float(r.loss) == float(want[k].loss)


def test_offsets_beyond_32_bits(ctx):
    """2.2e9 kept logits (4.5 GB), checked against 64 bits a thousand rows at a time."""
    bt, h, v = 17000, 64, 131072
    x, w, labels = make(bt, h, v, seed=51, ignored=0.1)
    r = call(ctx, x, w, labels, grad_dtype=torch.bfloat16, piece_bytes=8 << 30)
    live = labels != -100
    n = int(live.sum())
    wd = w.double()
    dw = torch.zeros(v, h, dtype=torch.float64, device="cuda")
    for rows in torch.arange(bt, device="cuda").split(1000):
        xd = torch.where(live[rows, None], x[rows].double(), 0.0)
        z = xd @ wd.T
        lse = torch.logsumexp(z, 1)
        y = torch.where(live[rows], labels[rows], 0)
        nll = torch.where(live[rows], lse - z.gather(1, y[:, None])[:, 0], 0.0)
        # logits of 64 products below 8 in magnitude: 2 H 2^-24 sum |h w| < 1e-4
        assert (r.nll[rows].double() - nll).abs().max() < 1e-4
        d = torch.exp(z - lse[:, None])
        d[torch.arange(len(rows), device="cuda"), y] -= 1
        d *= live[rows, None] / n
        dw += d.T @ xd
        dh = d @ wd
        assert (r.grad_hidden[rows].double() - dh).norm() < 1.6e-3 * math.sqrt(3) * dh.norm()
    assert (r.grad_weight.double() - dw).norm() < 1.6e-3 * math.sqrt(3) * dw.norm()


@pytest.mark.parametrize("bt", [64, 300])
@pytest.mark.parametrize("piece_bytes", [0, 1])
def test_label_at_the_lowest_value(ctx, bt, piece_bytes):
    """Labels on vocabulary entries that a large negative logit masks: z log2 e leaves fp32, the other entries'
    softmax does not."""
    x, w, labels = make(bt, 64, 640, seed=6)
    x[:, 0] = 1.0
    w[:, 0] = 0.0
    w[128:384, 0] = -3.0e38
    labels = torch.where((labels >= 128) & (labels < 384), 5, labels)
    labels[::3] = 200
    r = call(ctx, x, w, labels, mean=False, piece_bytes=piece_bytes)
    keep = torch.cat([torch.arange(128), torch.arange(384, 640)]).cuda()
    z = x.double() @ w[keep].double().T
    lse = torch.logsumexp(z, 1)
    f = formula(x, w[keep].contiguous(), torch.zeros(bt, dtype=torch.int64, device="cuda"))
    assert torch.all((r.lse.double() - lse).abs() <= f["row_tol"])
    masked = torch.zeros(bt, dtype=torch.bool, device="cuda")
    masked[::3] = True
    zy = (x.double() * w.double()[labels]).sum(1)
    # 2^-22 of a loss of 3e38: the products' sum and the difference to lse
    tol = f["row_tol"] + 2.0**-22 * zy.abs()
    assert torch.all((r.nll.double() - (lse - zy)).abs() <= tol)
    # the gradients: p over the entries that are left, -1 at the label
    p = torch.zeros(bt, 640, dtype=torch.float64, device="cuda")
    p[:, keep] = torch.exp(z - lse[:, None])
    p[torch.arange(bt, device="cuda"), labels] -= 1
    dw = p.T @ x.double()
    assert torch.isfinite(r.grad_hidden).all() and torch.isfinite(r.grad_weight).all()
    assert (r.grad_weight.double() - dw).norm() < 5e-3 * dw.norm()
    others = ~masked
    dh = p[others][:, keep] @ w[keep].double()
    assert (r.grad_hidden[others].double() - dh).norm() < 5e-3 * dh.norm()


@pytest.mark.parametrize("bt", [64, 300])
def test_a_row_of_lowest_values_only_shows(ctx, bt):
    x, w, labels = make(bt, 64, 640, seed=6)
    x[:, 0] = 0.0
    x[5, 0] = 1.0
    f = formula(x, w, labels)
    w[:, 0] = -3.0e38
    r = call(ctx, x, w, labels, need_grad_hidden=False, need_grad_weight=False)
    rest = torch.arange(bt, device="cuda") != 5
    assert torch.isnan(r.nll[5]) and torch.isnan(r.lse[5])
    g = formula(x[rest], w, labels[rest])
    tol = f["row_tol"][rest] + 2.0**-23 * g["nll"].abs()
    assert torch.all((r.nll[rest].double() - g["nll"]).abs() <= tol)


@pytest.mark.parametrize("bt", [20, 300])
@pytest.mark.parametrize("dense", [False, True])
def test_logits_whose_sums_are_exact(ctx, bt, dense):
    """Equal rows of weight and products that fp32 adds up without rounding: every logit is the same z, so lse - z =
    log V. fp32 rounds z log2 e and z (2^-24 of each, and twice more in lse), an exponential is off by 2^-22 and a sum
    of V of them by 2^-21 at most; the results round once more."""
    h, v = 4096, 5000
    x = torch.zeros(bt, h, device="cuda", dtype=torch.bfloat16)
    w = torch.zeros(v, h, device="cuda", dtype=torch.bfloat16)
    z = torch.tensor([100.0, -75.0, 50.0, 3.0, 0.0], device="cuda").repeat(bt)[:bt]
    if dense:
        w[:] = 2.0**-6
        x[:] = (z / 64).to(torch.bfloat16)[:, None]
        z = x[:, 0].double() * 64
    else:
        w[:, 0] = 1.0
        x[:, 0] = z.to(torch.bfloat16)
        z = z.double()
    labels = torch.arange(bt, device="cuda") * 7 % v
    for grads in (False, True):
        r = call(ctx, x, w, labels, need_grad_hidden=grads, need_grad_weight=grads, grad_dtype=torch.bfloat16)
        tol = 2 * 2.0**-24 * z.abs() + 2.0**-20 + 2.0**-22 * math.log(v)
        assert torch.all((r.nll.double() - math.log(v)).abs() <= tol), float((r.nll.double() - math.log(v)).abs().max())
        assert torch.all((r.lse.double() - math.log(v) - z).abs() <= 2 * tol)



@pytest.mark.parametrize("bt,h", [(64, 4096), (100, 4096), (300, 4096), (300, 2000), (300, 6200), (20, 9000)])
def test_logits_of_long_products_are_not_cut(ctx, bt, h):
    """Random operands: the tensor cores' sums over k come out too small by k 2^-30 of themselves on average, and the
    logits sum at most 2048 at once. lse is at most its largest logits and log V, so its mean relative error stays
    within 2048 2^-30 (twice to four times that where K is summed in one; the mean logit under the softmax is 0.93 of lse here) and
    that of the rounded results, 2^-24 / sqrt(bt)."""
    gen = torch.Generator(device="cuda").manual_seed(bt + h)
    v = 5003
    w = (torch.randn(v, h, generator=gen, device="cuda") * (6.0 / math.sqrt(h))).bfloat16()
    x = torch.randn(bt, h, generator=gen, device="cuda").bfloat16()
    labels = torch.randint(0, v, (bt,), generator=gen, device="cuda")
    lse = torch.logsumexp(x.double() @ w.double().T, 1)
    for grads in (False, True):
        r = call(ctx, x, w, labels, need_grad_hidden=grads, need_grad_weight=grads)
        off = float(((r.lse.double() - lse) / lse).mean())
        assert abs(off) <= 2048 * 2.0**-30 + 3 * 2.0**-24 / math.sqrt(bt), off


def test_a_refused_workspace_leaves_a_captured_one(ctx):
    """A workspace that a graph holds stays the context's when a larger one cannot be had (275 GB of statistics)."""
    from orda_b200.device import DeviceContext, linear_cross_entropy_device

    x, w, labels = make(100, 128, 2000, seed=11)
    with DeviceContext(0) as own:
        want = call(own, x, w, labels)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            r = linear_cross_entropy_device(own, x, w, labels)
        held = own.workspace_bytes()
        bt, v = 1 << 19, 1 << 22
        huge = [torch.zeros(bt, 8, device="cuda", dtype=torch.bfloat16),
                torch.zeros(v, 8, device="cuda", dtype=torch.bfloat16), torch.zeros(bt, device="cuda", dtype=torch.int64)]
        with pytest.raises(RuntimeError, match="workspace"):
            linear_cross_entropy_device(own, *huge, need_grad_hidden=False, need_grad_weight=False)
        assert own.workspace_bytes() == held
        second = torch.cuda.CUDAGraph()
        with torch.cuda.graph(second):
            r2 = linear_cross_entropy_device(own, x, w, labels)
        graph.replay()
        second.replay()
        torch.cuda.synchronize()
        own.check()
        assert torch.equal(r.grad_weight, want.grad_weight) and torch.equal(r2.grad_weight, want.grad_weight)
        del graph, second


def test_a_replay_leaves_a_vocabulary_forward_phase(ctx):
    """A captured call replayed between the two phases of a vocabulary-sharded step on the same context."""
    import orda_b200 as ob
    from orda_b200.device import (DeviceContext, linear_cross_entropy_device, vocab_backward_device,
                                  vocab_forward_device)

    x, w, labels = make(256, 128, 4096, seed=19)
    teacher = (x.float() * 0.9).bfloat16()
    opts = ob.LossOptions(kd_weight=0.4, temperature=1.5)
    big = make(400, 256, 9000, seed=20)
    with DeviceContext(0) as own:
        call(own, *big)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            r = linear_cross_entropy_device(own, *big)
        got = []
        for replay in (False, True):
            part = vocab_forward_device(own, x, w, labels, ob.TeacherMode.Tied, 4096, 0, opts=opts,
                                        teacher_hidden=teacher)
            if replay:
                graph.replay()
            got.append(vocab_backward_device(own, x, w, labels, ob.TeacherMode.Tied, 4096, 0, part[None], True,
                                             opts=opts, teacher_hidden=teacher))
        torch.cuda.synchronize()
        own.check()
        assert torch.equal(got[0].scalars, got[1].scalars)
        assert torch.equal(got[0].grad_weight, got[1].grad_weight)
        assert torch.equal(got[0].grad_student_hidden, got[1].grad_student_hidden)
        check(r, formula(*big))
        del graph


def test_faults_of_earlier_calls_are_reported(ctx):
    """A bad id and a bad label are reported one after the other; a distillation call's bad label and an expired
    wait outlive a cross entropy call, and what has been reported is not reported again after it."""
    import orda_b200 as ob
    from orda_b200 import _abi
    from orda_b200.device import DeviceContext, distillation_loss_device, embedding_device, linear_cross_entropy_device

    x, w, labels = make(40, 64, 300)
    bad = labels.clone()
    bad[7] = 300
    with DeviceContext(0) as own:
        embedding_device(own, w, bad)
        linear_cross_entropy_device(own, x, w, bad)
        linear_cross_entropy_device(own, x, w, labels)
        with pytest.raises(ob.OrdaError, match="token id"):
            own.check()
        with pytest.raises(ob.OrdaError, match="label is out of range"):
            own.check()
        own.check()
        # in the other order, and two of each: one report for each kind
        for _ in range(2):
            linear_cross_entropy_device(own, x, w, bad)
            embedding_device(own, w, bad)
        for _ in range(2):
            with pytest.raises(ob.OrdaError) as e:
                own.check()
            assert e.value.code == _abi.ORDA_ERR_LABEL
        own.check()
        # a distillation call keeps its state in a word of its own kind
        opts = ob.LossOptions(kd_weight=0.0, teacher_ce_weight=0.0)
        distillation_loss_device(own, x, w, bad, ob.TeacherMode.Tied, teacher_hidden=x, opts=opts)
        r = linear_cross_entropy_device(own, x, w, labels)
        with pytest.raises(ob.OrdaError, match="label is out of range"):
            own.check()
        own.check()
        check(r, formula(x, w, labels))
        # reported before the cross entropy call: not again after it
        distillation_loss_device(own, x, w, bad, ob.TeacherMode.Tied, teacher_hidden=x, opts=opts)
        with pytest.raises(ob.OrdaError, match="label is out of range"):
            own.check()
        check(call(own, x, w, labels), formula(x, w, labels))
        # an expired wait, likewise
        own.selftest_bounded_wait(1000)
        linear_cross_entropy_device(own, x, w, labels)
        with pytest.raises(ob.OrdaError) as e:
            own.check()
        assert e.value.code == _abi.ORDA_ERR_TIMEOUT
        own.check()
        own.selftest_bounded_wait(1000)
        with pytest.raises(ob.OrdaError):
            own.check()
        check(call(own, x, w, labels), formula(x, w, labels))


def test_smaller_pieces_are_kept_and_captured(ctx):
    """A call that took smaller pieces because memory was short can be captured, and neither it nor later calls
    ask for the larger workspace again."""
    from orda_b200.device import DeviceContext, linear_cross_entropy_device

    x, w, labels = make(64, 64, 3000, seed=14)
    with DeviceContext(0) as own:
        own.inject_alloc_failures(2)
        first = call(own, x, w, labels)
        held = own.workspace_bytes()
        again = call(own, x, w, labels)
        assert own.workspace_bytes() == held
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            r = linear_cross_entropy_device(own, x, w, labels)
        graph.replay()
        torch.cuda.synchronize()
        own.check()
        assert own.workspace_bytes() == held
        for n in ("loss", "nll", "lse", "grad_hidden", "grad_weight"):
            assert torch.equal(getattr(r, n), getattr(first, n)) and torch.equal(getattr(r, n), getattr(again, n)), n
        # a larger call for which no piece fits that workspace still gets its own
        big = make(300, 64, 9000, seed=15)
        check(call(own, *big), formula(*big))
        assert own.workspace_bytes() > held
        del graph


def test_few_rows_leave_no_kept_lines(ctx):
    """With the persisting-L2 carve-out on, a call of few tokens demotes the hidden copy too: one launch more."""
    from orda_b200.device import DeviceContext

    x, w, labels = make(8, 512, 5000, seed=17)
    counts, results = [], []
    for carve in (0, 64 << 20):
        with DeviceContext(0) as own:
            if carve:
                assert own.set_l2_persisting(carve) > 0
            call(own, x, w, labels, need_grad_hidden=False, need_grad_weight=False)
            n = own.launch_count()
            results.append(call(own, x, w, labels, need_grad_hidden=False, need_grad_weight=False))
            counts.append(own.launch_count() - n)
    assert counts[1] == counts[0] + 1
    assert torch.equal(results[0].nll, results[1].nll) and torch.equal(results[0].lse, results[1].lse)


def test_the_capture_stream_may_end(ctx):
    """A graph outlives the stream that it was captured on; check() then looks at no stream that is gone."""
    from cuda.bindings import runtime as rt

    from orda_b200.device import DeviceContext, embedding_device, embedding_grad_device, linear_cross_entropy_device

    def ok(res):
        assert int(res[0]) == 0, res
        return res[1] if len(res) > 1 else None

    x, w, labels = make(40, 64, 300, seed=18)
    out = {"loss": torch.zeros(1, device="cuda"), "nll": torch.zeros(40, device="cuda"),
           "lse": torch.zeros(40, device="cuda"), "grad_hidden": torch.zeros(40, 64, device="cuda"),
           "grad_weight": torch.zeros(300, 64, device="cuda")}
    rows, table = torch.zeros(40, 64, device="cuda"), torch.zeros(300, 64, device="cuda")
    steps = [lambda c, s: linear_cross_entropy_device(c, x, w, labels, out=out, stream=s),
             lambda c, s: embedding_device(c, w, labels, out=rows, stream=s),
             lambda c, s: embedding_grad_device(c, rows, labels, 300, scale=2.0, out=table, stream=s)]
    for step in steps:
        with DeviceContext(0) as own:
            step(own, None)
            torch.cuda.synchronize()
            s = ok(rt.cudaStreamCreateWithFlags(rt.cudaStreamNonBlocking))
            ok(rt.cudaStreamBeginCapture(s, rt.cudaStreamCaptureMode.cudaStreamCaptureModeThreadLocal))
            step(own, int(s))
            graph = ok(rt.cudaStreamEndCapture(s))
            run = ok(rt.cudaGraphInstantiate(graph, 0))
            ok(rt.cudaStreamDestroy(s))
            for t in (*out.values(), rows, table):
                t.fill_(7.0)
            ok(rt.cudaGraphLaunch(run, torch.cuda.current_stream().cuda_stream))
            torch.cuda.synchronize()
            own.check()
            ok(rt.cudaGraphExecDestroy(run))
            ok(rt.cudaGraphDestroy(graph))
            if step is steps[0]:
                f = formula(x, w, labels)
                assert torch.all((out["nll"].double() - f["nll"]).abs() <= f["row_tol"] + 2.0**-23 * f["nll"].abs())
            elif step is steps[1]:
                assert torch.equal(rows, w[labels].float())
            else:
                assert not (table == 7.0).any()


def test_phase_timing_and_capture(ctx):
    """A captured call leaves no events behind whose times could not be read."""
    from orda_b200.device import DeviceContext, linear_cross_entropy_device

    x, w, labels = make(150, 64, 900, seed=24)
    with DeviceContext(0) as own:
        own.enable_timing()
        call(own, x, w, labels)
        once = own.phase_times()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            linear_cross_entropy_device(own, x, w, labels)
        graph.replay()
        torch.cuda.synchronize()
        assert own.phase_times() == once
        check(call(own, x, w, labels), formula(x, w, labels))
        twice = own.phase_times()
        assert all(twice[k][1] == 2 * n and twice[k][0] >= ms for k, (ms, n) in once.items())
        del graph


def test_loss_of_certain_tokens(ctx):
    """Rows that are all but certain: the loss is the sum of the other entries' e^(z - z_label), each off by its
    logit's error (2 H 2^-24 sum |h w| = 8e-4 at H = 64 here) and an exponential's, none by a cancellation."""
    h, v = 64, 1200
    gen = torch.Generator(device="cuda").manual_seed(2)
    w = (torch.randn(v, h, generator=gen, device="cuda") * 0.1).bfloat16()
    w[:, 0] = -1.0
    w[-1, 0] = 1.0
    for bt in (4, 200):
        x = torch.zeros(bt, h, device="cuda", dtype=torch.bfloat16)
        x[:, 0] = torch.linspace(6, 40, bt, device="cuda").to(torch.bfloat16)
        x[:, 1:] = (torch.randn(bt, h - 1, generator=gen, device="cuda") * 0.1).bfloat16()
        labels = torch.full((bt,), v - 1, device="cuda")
        z = x.double() @ w.double().T
        want = torch.log1p(torch.exp(z[:, :-1] - z[:, -1:]).sum(1))
        ez = 2 * h * 2.0**-24 * (x.double().abs() @ w.double().abs().T).amax(1)
        # ... and 2^-24 of the exponent z log2 e, at the row's reference and in the sum
        tol = (2 * ez + 4 * 2.0**-24 * z.abs().amax(1) * 2 + 2.0**-20) * want
        for piece in (0, 1):
            r = call(ctx, x, w, labels, piece_bytes=piece)
            assert float(want.min()) > 1e-32 and float(want.max()) < 1e-1
            assert torch.all((r.nll.double() - want).abs() <= tol), float(((r.nll.double() - want).abs() / want).max())


@pytest.mark.parametrize("piece_bytes", [0, 1])
@pytest.mark.parametrize("bt", [300, 1100])
def test_far_labels_of_many_tokens(ctx, piece_bytes, bt):
    """As test_far_labels, with the logits of more tokens than the few-row kernel takes."""
    h, v = 64, 1200
    gen = torch.Generator(device="cuda").manual_seed(2)
    w = torch.zeros(v, h, device="cuda")
    w[:, 0] = torch.linspace(-1, 1, v, device="cuda")
    w[:, 1:] = torch.randn(v, h - 1, generator=gen, device="cuda") * 0.1
    w = w.bfloat16()
    x = torch.randn(bt, h, generator=gen, device="cuda")
    x[:, 0] = torch.linspace(-150, 150, bt, device="cuda")
    x = x.bfloat16()
    labels = torch.randint(0, v, (bt,), generator=gen, device="cuda")
    labels[::3] = 0
    labels[1::3] = v - 1
    f = formula(x, w, labels)
    check(call(ctx, x, w, labels, grad_dtype=torch.bfloat16, piece_bytes=piece_bytes), f)
    check(call(ctx, x, w, labels, need_grad_hidden=False, need_grad_weight=False), f)
    f = formula(x, w, labels, 0.1)
    check(call(ctx, x, w, labels, 0.1, grad_dtype=torch.bfloat16, piece_bytes=piece_bytes), f)


@pytest.mark.parametrize("piece_bytes", [0, 1])
def test_lowest_value_logits_of_many_tokens(ctx, piece_bytes):
    x, w, labels = make(300, 64, 640, seed=6)
    x[:, 0] = 1.0
    w[:, 0] = 0.0
    w[128:384, 0] = -3.0e38
    labels[(labels >= 128) & (labels < 384)] = 5
    r = call(ctx, x, w, labels, grad_dtype=torch.bfloat16, piece_bytes=piece_bytes)
    keep = torch.cat([torch.arange(128), torch.arange(384, 640)]).cuda()
    sub = torch.full((640,), 0, device="cuda")
    sub[keep] = torch.arange(len(keep), device="cuda")
    f = formula(x, w[keep].contiguous(), sub[labels])
    assert torch.all((r.nll.double() - f["nll"]).abs() <= f["row_tol"])
    assert not r.grad_weight[128:384].any()
    assert ((r.grad_weight[keep].double() - f["dw"]).norm() / f["dw"].norm()) < 5e-3


@pytest.mark.parametrize("piece_bytes", [0, 1])
def test_nan_of_a_live_row_of_many_shows(ctx, piece_bytes):
    x, w, labels = make(300, 64, 1300)
    x[133, 5] = float("nan")
    r = call(ctx, x, w, labels, piece_bytes=piece_bytes)
    assert torch.isnan(r.loss) and torch.isnan(r.nll[133]) and torch.isnan(r.grad_hidden[133]).all()
    rest = [i for i in range(300) if i != 133]
    assert torch.isfinite(r.nll[rest]).all() and torch.isfinite(r.grad_hidden[rest]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_wide_weight_gradient_tiles(ctx, dtype):
    """8200 tokens: a K loop long enough for the 256 x 512 tiles of grad_weight. Relative L2 as in
    test_larger_products."""
    x, w, labels = make(8200, 512, 38005, seed=23, ignored=0.1)
    r = call(ctx, x, w, labels, grad_dtype=dtype)
    live = labels != -100
    n = int(live.sum())
    wd, dw = w.double(), torch.zeros(38005, 512, dtype=torch.float64, device="cuda")
    for rows in torch.arange(8200, device="cuda").split(2050):
        xd = torch.where(live[rows, None], x[rows].double(), 0.0)
        d = torch.softmax(xd @ wd.T, 1)
        d[torch.arange(len(rows), device="cuda"), torch.where(live[rows], labels[rows], 0)] -= 1
        d *= live[rows, None] / n
        dw += d.T @ xd
        dh = d @ wd
        assert (r.grad_hidden[rows].double() - dh).norm() < 1.6e-3 * math.sqrt(3) * dh.norm()
    assert (r.grad_weight.double() - dw).norm() < 1.6e-3 * math.sqrt(3) * dw.norm()


@pytest.mark.parametrize("env", [{"ORDA_GEMM_CTA_PAIR": "0"}, {"ORDA_GEMM_WIDE": "2"}])
@pytest.mark.parametrize("bt,h,v", [(300, 520, 4099), (260, 2200, 1500)])
def test_other_tiles(ctx, monkeypatch, env, bt, h, v):
    """Single-CTA tiles, and 256 x 512 ones wherever they can be; K in one part and in two."""
    for k, val in env.items():
        monkeypatch.setenv(k, val)
    x, w, labels = make(bt, h, v, seed=25, ignored=0.1)
    for a, piece in ((0.0, 0), (0.1, bt * 1024 * 2)):
        f = formula(x, w, labels, a)
        for dtype in (torch.float32, torch.bfloat16):
            check(call(ctx, x, w, labels, a, grad_dtype=dtype, piece_bytes=piece), f)
        check(call(ctx, x, w, labels, a, need_grad_hidden=False, need_grad_weight=False), f)


@pytest.mark.parametrize("bt", [70, 300])
@pytest.mark.parametrize("h", [2048, 2056, 4096, 4160])
def test_long_rows(ctx, bt, h):
    """K of the logits in one, two and three parts, with labels far above, far below and among the others."""
    x, w, labels = make(bt, h, 1201, seed=h, ignored=0.1)
    w[:, 0] = 0.0
    w[:600, 0] = 1.0
    x[:, 0] = torch.linspace(-100, 100, bt, device="cuda").to(torch.bfloat16)
    # In the part where the two groups of entries meet the fixed point holds a probability as zero that is at most
    # 2^-64 of its reference's, the label's or one of the part's: at most 2^-64. Elsewhere such probabilities count.
    live = labels != -100
    p = torch.where(live[:, None], torch.softmax(x.double() @ w.double().T, 1), 0.0)
    p = torch.where(p <= 2.0**-64, p, 0.0)[:, 576:640] / int(live.sum())
    for a in (0.0, 0.1):
        f = formula(x, w, labels, a)
        f["dh_tol"] += p @ w[576:640].double().abs()
        f["dw_tol"][576:640] += p.T @ x.double().abs()
        for piece in (0, 1):
            check(call(ctx, x, w, labels, a, piece_bytes=piece), f)
        check(call(ctx, x, w, labels, a, need_grad_hidden=False, need_grad_weight=False), f)


def test_checks_from_another_thread(ctx):
    """check() beside calls of the same context: every bad call is heard of, the good calls' results stand."""
    import threading

    import orda_b200 as ob
    from orda_b200.device import DeviceContext, distillation_loss_device, linear_cross_entropy_device

    x, w, labels = make(150, 64, 900, seed=26)
    bad = labels.clone()
    bad[3] = 900
    opts = ob.LossOptions(kd_weight=0.0, teacher_ce_weight=0.0)
    with DeviceContext(0) as own:
        want = call(own, x, w, labels)
        stop, heard, other = threading.Event(), [], []

        def listen():
            while not stop.is_set():
                try:
                    own.check()
                except ob.OrdaError as e:
                    (heard if "label is out of range" in str(e) else other).append(str(e))

        thread = threading.Thread(target=listen)
        thread.start()
        results = []
        for i in range(60):
            if i % 10 == 0:
                distillation_loss_device(own, x, w, bad, ob.TeacherMode.Tied, teacher_hidden=x, opts=opts)
            results.append(linear_cross_entropy_device(own, x, w, labels))
        torch.cuda.synchronize()
        stop.set()
        thread.join()
        try:
            own.check()
        except ob.OrdaError as e:
            heard.append(str(e))
        own.check()
        assert heard and not other
        for r in results:
            assert torch.equal(r.grad_weight, want.grad_weight) and float(r.loss) == float(want.loss)
