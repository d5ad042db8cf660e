"""The operators beside the programs on the GPU, against plain forms in 64 bits.

Tolerances count roundings: half a step of the result's type, relative to the result; f32 sums one rounding (2^-24) a term,
relative to the sum of magnitudes; weights of the attention one rounding of the type they are multiplied in."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from conftest import package  # noqa: E402
from operator_refs import DT, U, Paged, half_step, normal, quantised, rope  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rt():
    r = package().Runtime.Create(0)
    yield r
    r.close()


@pytest.fixture(scope="module")
def scratch(rt):
    s = package().Scratch.Create(rt)
    yield s
    s.close()


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _views(n, hq, hk, dim, dtype, layout, seed, scale=1.0):
    """Queries and keys: views of a fused projection, heads first, or a copy whose rows start one element off any alignment."""
    qkv = normal((n, (hq + 2 * hk) * dim), dtype, seed, scale)
    q, k = qkv[:, :hq * dim].view(n, hq, dim), qkv[:, hq * dim:(hq + hk) * dim].view(n, hk, dim)
    if layout == "heads_first":
        return tuple(x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k))
    if layout == "odd":
        out = []
        for x in (q, k):
            flat = torch.empty(x.numel() + 3 * n + 1, dtype=x.dtype, device="cuda")
            y = flat[1:].as_strided(x.shape, (x.shape[1] * dim + 3, dim, 1), 1)
            y.copy_(x)
            out.append(y)
        return tuple(out)
    return q, k


ROPE = [  # rows, q heads, k heads, dim, rot, dtype, interleaved, norm, layout, weights, scaling
    (1, 16, 16, 64, 64, "bf16", False, False, "fused", None, "plain"),
    (33, 32, 8, 128, 128, "bf16", False, True, "fused", "f32", "parts"),
    (7, 5, 1, 128, 64, "f16", True, True, "heads_first", "rows", "linear"),
    (129, 3, 2, 96, 48, "f32", True, True, "fused", "f32", "stretch"),
    (20, 4, 4, 80, 80, "bf16", False, True, "odd", "f32", "plain"),
    (5, 2, 1, 256, 256, "f16", False, False, "odd", None, "plain"),
    (11, 3, 0, 34, 30, "f32", False, True, "odd", None, "plain"),
    (6, 1, 3, 2, 2, "f32", True, False, "fused", None, "plain"),
    (300, 7, 7, 64, 0, "bf16", False, True, "fused", "rows", "plain"),
    (2500, 4, 2, 128, 96, "bf16", True, True, "fused", "f32", "plain"),
    (9, 2, 2, 200, 8, "f16", False, True, "heads_first", "f32", "plain"),
    (5001, 2, 1, 128, 128, "bf16", False, True, "fused", "f32", "plain"),        # (more than one token to a CTA, the last run shorter)
    (40, 3, 2, 256, 256, "bf16", False, True, "fused", "f32", "plain"),
    (17, 2, 2, 256, 128, "f32", True, True, "odd", "f32", "plain"),
    (16384 + 5, 1, 1, 64, 32, "f16", True, True, "fused", "f32", "plain"),
]


def _rope_case(rt, c, seed):
    vm = package()
    n, hq, hk, dim, rot, dtype, inter, norm, layout, weights, scaling = c
    freq = vm.RopeFrequencies(rot, 10000.0, scaling, 1.0 if scaling == "plain" else 4.0, 4096.0)
    mag = 1.25 if scaling == "parts" else 1.0
    wdt = dtype if weights == "rows" else "f32"
    handle = vm.Rope.Create(rt, head_dim=dim, rot_dim=rot, q_heads=hq, k_heads=hk, dtype=dtype, frequencies=freq, interleaved=inter, norm=norm, eps=1e-5,
                            weight_dtype=wdt, magnitude=mag)
    q, k = _views(n, hq, max(hk, 1), dim, dtype, layout, seed, 1.5)
    k = k[:, :hk]
    w = [(1.0 + 0.3 * normal((dim,), "f32", seed + 5 + i)).to(DT[wdt]) for i in range(2)] if weights else [None, None]
    pos = torch.randint(0, 200000, (n,), generator=torch.Generator().manual_seed(seed), dtype=torch.int32).cuda()
    pos[0] = 2 ** 31 - 1
    if n > 2:
        pos[1], pos[2] = 0, -5
    ref = lambda x, wt: rope(x, wt, pos, freq, rot, inter, norm, 1e-5, mag)  # noqa: E731
    return handle, q, k, w, pos, ref, mag


def _rows(t):
    return package().Rows.Of(t) if t.shape[1] else None


def _ptr(t):
    return 0 if t is None else t.data_ptr()


@pytest.mark.parametrize("c", ROPE, ids=lambda c: "-".join(map(str, c)))
def test_rotary_positions(rt, c):
    n, hq, hk, dim, rot, dtype, _, norm = c[:8]
    handle, q, k, w, pos, ref, mag = _rope_case(rt, c, 1)
    outs = [torch.full((n, h, dim), 7.0, dtype=DT[dtype], device="cuda") for h in (hq, hk)]
    handle.Apply(n, pos.data_ptr(), _rows(q), _rows(k), _rows(outs[0]), _rows(outs[1]), _ptr(w[0]), _ptr(w[1]), stream=_stream())
    for x, wt, out in zip((q, k), w, outs):
        want = ref(x.double(), wt.double() if wt is not None else None)
        # a pair's values: the norm (dim / 2 roundings of its sum, and 6), sine and cosine (4), two products and a sum; both of a pair count
        size = torch.ones_like(want)
        if norm:
            size = torch.rsqrt((x.double() ** 2).mean(-1, keepdim=True) + 1e-5) * (wt.double().abs().max() if wt is not None else 1.0)
        reach = 2 * x.double().abs().amax(-1, keepdim=True) * size * mag if x.numel() else size
        tol = half_step(dtype) * want.abs() + (dim / 2 + 20) * U * reach
        assert bool(((out.double() - want).abs() <= tol).all())
    # over its own inputs
    handle.Apply(n, pos.data_ptr(), _rows(q), _rows(k), _rows(q), _rows(k), _ptr(w[0]), _ptr(w[1]), stream=_stream())
    assert torch.equal(q, outs[0]) and torch.equal(k, outs[1])


@pytest.mark.parametrize("c", ROPE, ids=lambda c: "-".join(map(str, c)))
def test_rotary_positions_backward(rt, scratch, c):
    n, hq, hk, dim, rot, dtype, _, norm = c[:8]
    handle, q, k, w, pos, ref, mag = _rope_case(rt, c, 2)
    dy = list(_views(n, hq, max(hk, 1), dim, dtype, c[8], 9))
    dy[1] = dy[1][:, :hk]
    want_dw = norm and c[9] is not None
    grads, weights = [], []
    for turn in range(2):
        dx = [torch.empty((n, h, dim), dtype=DT[dtype], device="cuda") for h in (hq, hk)]
        dw = [torch.full((dim,), 3.0, device="cuda") if h else None for h in (hq, hk)] if want_dw else [None, None]
        handle.ApplyBackward(n, pos.data_ptr(), _rows(q) if norm else None, _rows(k) if norm else None, _rows(dy[0]), _rows(dy[1]), _rows(dx[0]), _rows(dx[1]),
                             _ptr(w[0]), _ptr(w[1]), _ptr(dw[0]), _ptr(dw[1]), scratch, stream=_stream())
        grads.append(dx)
        weights.append(dw)
    for i, x in enumerate((q, k)):
        if not x.shape[1]:
            continue
        leaf = x.double().requires_grad_()
        wt = (w[i].double() if w[i] is not None else torch.ones(dim, dtype=torch.float64, device="cuda")).requires_grad_()
        g = torch.autograd.grad(ref(leaf, wt), [leaf, wt], dy[i].double(), allow_unused=True)
        size = torch.rsqrt((x.double() ** 2).mean(-1, keepdim=True) + 1e-5) if norm else torch.ones_like(x[..., :1]).double()
        turned = 2 * dy[i].double().abs().amax(-1, keepdim=True) * mag * (wt.detach().abs().max() if norm else 1.0)
        xr = x.double().abs().amax(-1, keepdim=True) * size
        # r h - x r^3 mean(h x): the second sum has dim terms below |turned| |x|, its factors dim / 2 roundings of the norm thrice
        tol = half_step(dtype) * g[0].abs() + (3 * dim + 40) * U * turned * size * (1 + xr * xr if norm else 1.0)
        assert bool(((grads[0][i].double() - g[0]).abs() <= tol).all())
        assert torch.equal(grads[0][i], grads[1][i])
        if want_dw:
            terms = (turned / wt.detach().abs().max() * xr).sum((0, 1))
            assert bool(((weights[0][i].double() - g[1]).abs() <= (dim + n / 4 + 60) * U * terms).all())
            assert torch.equal(weights[0][i], weights[1][i])


@pytest.mark.parametrize("inter, rot", [(False, 64), (True, 32)])
def test_rotary_gradients_against_differences(rt, scratch, inter, rot):
    """Central differences of the forward pass itself, at h and h / 2: what the second is off by is below what halving changed, plus
    the roundings of the sums over the step."""
    vm = package()
    n, h, dim = 37, 3, 64
    handle = vm.Rope.Create(rt, head_dim=dim, rot_dim=rot, q_heads=h, k_heads=0, dtype="f32", interleaved=inter, norm=True, eps=1e-3)
    x, dy, v = (normal((n, h, dim), "f32", s) for s in (1, 2, 3))
    w, vw = 1.0 + 0.1 * normal((dim,), "f32", 4), normal((dim,), "f32", 5)
    pos = torch.arange(n, dtype=torch.int32, device="cuda") * 13

    def f(x, w):
        out = torch.empty_like(x)
        handle.Apply(n, pos.data_ptr(), _rows(x), None, _rows(out), None, w.data_ptr(), stream=_stream())
        return float((out.double() * dy.double()).sum()), float((out.double() * dy.double()).abs().sum())

    dx, dw = torch.empty_like(x), torch.empty_like(w)
    handle.ApplyBackward(n, pos.data_ptr(), _rows(x), None, _rows(dy), None, _rows(dx), None, w.data_ptr(), 0, dw.data_ptr(), 0, scratch, stream=_stream())
    for dirx, dirw, got in ((v, torch.zeros_like(vw), float((dx.double() * v.double()).sum())), (torch.zeros_like(v), vw, float((dw.double() * vw.double()).sum()))):
        d = []
        for step in (2.0 ** -5, 2.0 ** -6):
            (a, s), (b, _) = f(x + step * dirx, w + step * dirw), f(x - step * dirx, w - step * dirw)
            d.append((a - b) / (2 * step))
        assert abs(d[1] - got) <= abs(d[0] - d[1]) + (dim + 40) * U * s / 2.0 ** -6


def test_rotary_positions_of_nothing(rt, scratch):
    vm = package()
    handle = vm.Rope.Create(rt, head_dim=64, q_heads=2, k_heads=2, dtype="bf16", norm=True)
    handle.Apply(0, 0, None, None, None, None, stream=_stream())
    dw = torch.ones(2, 64, device="cuda")
    handle.ApplyBackward(0, 0, None, None, None, None, None, None, dq_weight=dw[0].data_ptr(), dk_weight=dw[1].data_ptr(), scratch=scratch, stream=_stream())
    assert not bool(dw.any())
    # a row of zeros without eps is 0 / 0 in its own row, and in no other's
    handle = vm.Rope.Create(rt, head_dim=64, q_heads=3, k_heads=0, dtype="f32", norm=True, eps=0.0)
    x = normal((5, 3, 64), "f32", 1)
    x[2, 1] = 0.0
    out, pos = torch.empty_like(x), torch.arange(5, dtype=torch.int32, device="cuda")
    handle.Apply(5, pos.data_ptr(), _rows(x), None, _rows(out), None, stream=_stream())
    bad = ~torch.isfinite(out).all(-1)
    assert bool(bad[2, 1]) and int(bad.sum()) == 1


CACHE = [  # rows, past, dtype, row dtype, heads, dim, page, head major, pad
    ([1, 1, 1], [0, 15, 16], "e4m3", "bf16", 2, 64, 16, False, 0),
    ([5, 0, 33, 1], [3, 7, 100, 0], "e4m3", "f16", 3, 128, 7, True, 6),
    ([40], [0], "e4m3", "f32", 1, 80, 1, False, 1),
    ([9, 70], [50, 2], "bf16", "bf16", 2, 128, 24, True, 0),
    ([17, 3], [1, 1000], "f16", "f32", 5, 16, 64, False, 40),
    ([1] * 40 + [0] * 3 + [2] * 40, [3] * 83, "e4m3", "bf16", 1, 48, 5, False, 3),
    ([2600, 1300], [5, 0], "e4m3", "bf16", 4, 128, 128, False, 9),
    ([3000], [70], "bf16", "f32", 8, 64, 32, False, 0),
    ([5000, 3, 2308], [1, 0, 9], "e4m3", "bf16", 1, 64, 64, False, 2),
    ([9001, 6000, 1, 4000], [0, 3, 50, 1], "f16", "f16", 2, 32, 16, False, 1),
]


@pytest.mark.parametrize("c", CACHE, ids=lambda c: f"{len(c[0])}x{max(c[0])}-" + "-".join(map(str, c[2:])))
@pytest.mark.parametrize("odd", [False, True])
def test_cache_written_and_read_back(rt, c, odd):
    rows, past, dtype, row_dtype, heads, dim, page, major, pad = c
    p = Paged(rt, rows, past, dtype=dtype, row_dtype=row_dtype, heads=heads, dim=dim, page=page, head_major=major, pad=pad)
    kv = [normal((p.n_rows, heads, dim), row_dtype, 20 + i, 3.0) for i in range(2)]
    kv[0][0] = 0.0
    if odd:                                                      # rows that start one element off any alignment
        for i in range(2):
            flat = torch.empty(kv[i].numel() + 1, dtype=kv[i].dtype, device="cuda")
            flat[1:].copy_(kv[i].flatten())
            kv[i] = flat[1:].view(kv[i].shape)
    want = [x.clone() for x in p.pages]
    scales = [s.clone() if s is not None else None for s in p.scales]
    at = torch.tensor(p.places(), device="cuda").long().reshape(-1, 3)
    back = []
    for i in range(2):
        x = kv[i][at[:, 0]]
        if dtype == "e4m3":
            codes, s = quantised(x.float())
            want[i].view(torch.uint8)[at[:, 1], at[:, 2]] = codes.view(torch.uint8)
            scales[i][at[:, 1], at[:, 2]] = s
            back.append((codes.float() * s[..., None]).to(DT[row_dtype]))
        else:
            want[i][at[:, 1], at[:, 2]] = x.to(DT[dtype])
            back.append(x.to(DT[dtype]).to(DT[row_dtype]))
    p.cache.Write(p.batch, package().Rows.Of(kv[0]), package().Rows.Of(kv[1]), stream=_stream())
    out = [torch.full((p.n_rows, heads, dim), 5.0, dtype=DT[row_dtype], device="cuda") for _ in range(2)]
    p.cache.Read(p.batch, package().Rows.Of(out[0]), package().Rows.Of(out[1]), stream=_stream())
    assert p.cache.Status()["code"] == 0
    for i in range(2):
        # bit for bit: both are divisions of f32 and one rounding
        assert torch.equal(p.pages[i].contiguous().view(torch.uint8), want[i].contiguous().view(torch.uint8))
        if dtype == "e4m3":
            assert torch.equal(p.scales[i], scales[i])
        assert torch.equal(out[i][at[:, 0]], back[i])
        assert bool((out[i][p.total:] == 5.0).all())             # rows behind the last sequence


def test_rows_that_are_not_finite_read_back_as_nan(rt):
    p = Paged(rt, [6], [10], dtype="e4m3", heads=1, dim=64)
    kv = [normal((6, 1, 64), "bf16", i) for i in range(2)]
    kv[0][1, 0, 5], kv[0][2, 0, 63], kv[1][4, 0, 0] = float("nan"), float("inf"), float("-inf")
    p.cache.Write(p.batch, package().Rows.Of(kv[0]), package().Rows.Of(kv[1]), stream=_stream())
    out = [torch.empty_like(x) for x in kv]
    p.cache.Read(p.batch, package().Rows.Of(out[0]), package().Rows.Of(out[1]), stream=_stream())
    assert [bool(torch.isnan(out[0][i]).all()) for i in range(6)] == [False, True, True, False, False, False]
    assert bool(torch.isfinite(out[0][[0, 3, 4, 5]]).all())
    assert bool(torch.isnan(out[1][4]).all()) and bool(torch.isfinite(out[1][[0, 1, 2, 3, 5]]).all())


def test_more_rows_than_positions(rt, scratch):
    """The rows before position 0 are not written, read as zeros and attend to nothing."""
    for rows, q_heads in ((5, 2), (40, 8)):
        p = Paged(rt, [rows, 2], [0, 3], lengths=[3, 5], dtype="bf16", heads=2, q_heads=q_heads, dim=64)
        before = [x.clone() for x in p.pages]
        kv = [normal((p.n_rows, 2, 64), "bf16", i) for i in range(2)]
        p.cache.Write(p.batch, package().Rows.Of(kv[0]), package().Rows.Of(kv[1]), stream=_stream())
        at = torch.tensor(p.places(), device="cuda").long()
        assert len(at) == 5
        for i in range(2):
            before[i][at[:, 1], at[:, 2]] = kv[i][at[:, 0]]
            assert torch.equal(before[i], p.pages[i])
        out = [torch.full_like(x, 5.0) for x in kv]
        p.cache.Read(p.batch, package().Rows.Of(out[0]), package().Rows.Of(out[1]), stream=_stream())
        assert not bool(out[0][:rows - 3].any()) and torch.equal(out[0][rows - 3:], kv[0][rows - 3:])
        q = normal((p.n_rows, q_heads, 64), "bf16", 5)
        o, lse = torch.full_like(q, 9.0), torch.zeros(p.n_rows, q_heads, device="cuda")
        p.cache.Attend(p.batch, package().Rows.Of(q), package().Rows.Of(o), scratch, lse=lse.data_ptr(), stream=_stream())
        want, want_lse, tol = p.attend(q, 64 ** -0.5)
        assert not bool(o[:rows - 3].any()) and bool((lse[:rows - 3] == float("-inf")).all())
        assert bool(((o.double() - want).abs() <= tol + half_step("bf16") * want.abs()).all())
        assert p.cache.Status()["code"] == 0


ATTEND = [  # rows, past, dtype, row dtype, heads, q heads, dim, page, causal, window, head major, pad
    ([1], [0], "bf16", "bf16", 1, 1, 64, 16, True, 0, False, 0),
    ([1], [300], "bf16", "bf16", 8, 32, 128, 64, True, 0, False, 0),
    ([1, 1, 1, 1], [0, 15, 16, 2000], "f16", "f16", 2, 14, 128, 7, True, 0, True, 2),
    ([1, 0, 1, 1], [5000, 9, 31, 700], "e4m3", "bf16", 2, 16, 128, 64, True, 0, False, 0),
    ([1] * 300, list(range(300)), "e4m3", "f16", 1, 4, 64, 16, True, 0, False, 0),
    ([4, 1, 3], [100, 0, 77], "bf16", "bf16", 2, 8, 80, 24, True, 0, False, 1),
    ([16], [333], "e4m3", "bf16", 3, 3, 64, 1, True, 20, True, 0),
    ([2, 1], [64, 5], "f16", "f16", 1, 5, 16, 3, False, 0, False, 0),
    ([1], [9000], "e4m3", "bf16", 1, 1, 48, 256, True, 4000, False, 0),
    ([17], [0], "bf16", "bf16", 1, 1, 64, 16, True, 0, False, 0),
    ([128], [128], "bf16", "bf16", 2, 2, 128, 64, True, 0, False, 0),
    ([129, 1, 0, 300], [70, 4000, 5, 0], "bf16", "bf16", 2, 8, 128, 48, True, 0, False, 5),
    ([200, 77], [31, 600], "e4m3", "bf16", 2, 10, 128, 64, True, 0, True, 0),
    ([260], [1500], "e4m3", "f16", 1, 7, 64, 24, True, 100, False, 0),
    ([90, 33], [10, 200], "f16", "f16", 4, 4, 80, 16, False, 0, False, 3),
    ([700], [0], "f16", "f16", 2, 2, 64, 5, True, 64, True, 0),
    ([1000], [3000], "bf16", "bf16", 1, 8, 128, 128, True, 0, False, 0),
    ([64] * 9, [0, 1, 63, 64, 65, 127, 128, 129, 1000], "f16", "f16", 1, 2, 96, 32, True, 0, False, 0),
    ([300], [2000], "e4m3", "bf16", 4, 4, 32, 16, True, 0, False, 0),
    # more tiles of rows than SMs: keys are not split
    ([600, 1, 90], [300, 777, 0], "bf16", "bf16", 16, 64, 128, 64, True, 0, False, 3),
    ([70] * 40, list(range(0, 800, 20)), "e4m3", "bf16", 4, 16, 128, 48, True, 0, True, 0),
    ([20] * 150, [37] * 150, "f16", "f16", 1, 2, 64, 16, True, 30, False, 0),
    ([513] * 3, [0, 100, 1000], "e4m3", "f16", 20, 20, 64, 32, True, 0, False, 0),
    ([40] * 30, [200] * 30, "bf16", "bf16", 5, 5, 80, 64, False, 0, False, 0),
]


@pytest.mark.parametrize("c", ATTEND, ids=lambda c: f"{len(c[0])}x{max(c[0])}-" + "-".join(map(str, c[2:])))
def test_attention_over_the_cache(rt, scratch, c):
    rows, past, dtype, row_dtype, heads, q_heads, dim, page, causal, window, major, pad = c
    p = Paged(rt, rows, past, dtype=dtype, row_dtype=row_dtype, heads=heads, q_heads=q_heads, dim=dim, page=page, head_major=major, pad=pad, seed=3)
    q = normal((p.n_rows, q_heads, dim), row_dtype, 8, 2.0)
    scale = dim ** -0.5
    want, want_lse, tol = p.attend(q, scale, causal, window)
    # a score's dim roundings (at most 16 x sum |q k| / dim here: below 2^-19), the sum's, and one of the result
    lse_tol = 2.0 ** -19 * (1 + want_lse.abs())
    for turn in range(2):                                        # (the second call finds the counters as the first left them)
        o, lse = torch.full_like(q, 9.0), torch.full((p.n_rows, q_heads), 9.0, device="cuda")
        p.cache.Attend(p.batch, package().Rows.Of(q), package().Rows.Of(o), scratch, lse=lse.data_ptr(), causal=causal, window=window, stream=_stream())
        assert p.cache.Status()["code"] == 0
        assert bool(((o[:p.total].double() - want).abs() <= tol + half_step(row_dtype) * want.abs()).all())
        assert bool(((lse[:p.total].double() - want_lse).abs() <= lse_tol).all())
        assert bool((o[p.total:] == 9.0).all()) and bool((lse[p.total:] == 9.0).all())
        if turn:
            assert torch.equal(o, first)
        first = o
    # without lse, heads first, one element off any alignment
    flat = torch.full((p.n_rows * q_heads * dim + 1,), 9.0, dtype=q.dtype, device="cuda")
    o2 = flat[1:].view(q_heads, p.n_rows, dim).transpose(0, 1)
    q2 = torch.empty_like(flat)[1:].view(q_heads, p.n_rows, dim).transpose(0, 1)
    q2.copy_(q)
    p.cache.Attend(p.batch, package().Rows.Of(q2), package().Rows.Of(o2), scratch, causal=causal, window=window, stream=_stream())
    assert torch.equal(o2, first)


@pytest.mark.parametrize("dtype, rows, past, q_heads, window, dim", [
    ("bf16", 4, 40, 4, 0, 64), ("e4m3", 8, 30, 2, 5, 128), ("f16", 70, 61, 4, 0, 64), ("bf16", 300, 5, 2, 33, 128), ("e4m3", 140, 0, 6, 0, 64), ("e4m3", 130, 300, 2, 50, 128)])
def test_what_a_row_does_not_see_does_not_reach_it(rt, scratch, dtype, rows, past, q_heads, window, dim):
    """A NaN, an infinity or a very large value at position c shows in the rows that see c and in no other; so does nothing that lies
    in the slots behind a sequence's end."""
    p = Paged(rt, [rows, 1], [past, 20], dtype=dtype, heads=1, q_heads=q_heads, dim=dim, page=16, seed=5)
    q = normal((p.n_rows, q_heads, dim), p.row_dtype, 8)
    want, _, tol = p.attend(q, dim ** -0.5, True, window)
    tol = tol + half_step(p.row_dtype) * want.abs()
    length = rows + past
    vm = package()
    # everything that is nobody's position is made NaN
    mine = torch.zeros(p.n_pages, p.page, dtype=torch.bool, device="cuda")
    for b in range(2):
        pos = torch.arange(p.lengths[b], device="cuda")
        mine[p.table[b, pos // p.page].long(), pos % p.page] = True
    for i in range(2):
        if dtype == "e4m3":
            p.pages[i].view(torch.uint8)[~mine] = 0x7F
            p.scales[i][~mine] = float("nan")
        else:
            p.pages[i][~mine] = float("nan")
    clean = [x.clone() for x in p.pages], [s.clone() if s is not None else None for s in p.scales]
    row = torch.arange(length - rows, length, device="cuda")
    for c in sorted({length - 1, length - 2, past, past + 1, max(0, past - 2), length - rows // 2}):
        for value in (float("nan"), float("inf"), "large"):
            for i in range(2):
                p.pages[i].copy_(clean[0][i])
                if dtype == "e4m3":
                    p.scales[i].copy_(clean[1][i])
            page, slot = int(p.table[0, c // 16]), c % 16
            if dtype == "e4m3":
                p.scales[1][page, slot] = 1e30 if value == "large" else value
                if value == "large":
                    p.pages[1].view(torch.uint8)[page, slot] = 0x7E
            else:
                p.pages[1][page, slot] = torch.finfo(DT[dtype]).max if value == "large" else value
                if value != "large":
                    p.pages[0][page, slot] = value
            o = torch.empty_like(q)
            p.cache.Attend(p.batch, vm.Rows.Of(q), vm.Rows.Of(o), scratch, window=window, stream=_stream())
            sees = (c <= row) & ((c > row - window) if window else True)
            got = o[:rows]
            ok = ((got.double() - want[:rows]).abs() <= tol[:rows]).all(-1).all(-1)
            assert bool(ok[~sees].all()), (c, value)
            assert bool(((o[rows:].double() - want[rows:]).abs() <= tol[rows:]).all())
            if value != "large":
                assert not bool(torch.isfinite(got[sees]).any()), (c, value)


@pytest.mark.parametrize("rows, q_heads", [(1, 4), (2, 8), (5, 2), (60, 4)])
def test_rows_of_zeros_in_an_8_bit_cache(rt, scratch, rows, q_heads):
    """Their scale is 0: all of the cache, its first positions, its last ones."""
    vm = package()
    for zeros in (slice(0, None), slice(0, 40), slice(90, None)):
        p = Paged(rt, [rows], [100], dtype="e4m3", heads=2, q_heads=q_heads, dim=64, page=16, seed=9)
        pos = torch.arange(100 + rows, device="cuda")[zeros]
        for i in range(2):
            p.pages[i].view(torch.uint8)[p.table[0, pos // 16].long(), pos % 16] = 0
            p.scales[i][p.table[0, pos // 16].long(), pos % 16] = 0.0
        q = normal((rows, q_heads, 64), "bf16", 8, 2.0)
        o = torch.empty_like(q)
        p.cache.Attend(p.batch, vm.Rows.Of(q), vm.Rows.Of(o), scratch, stream=_stream())
        want, _, tol = p.attend(q, 0.125)
        assert bool(((o.double() - want).abs() <= tol + half_step("bf16") * want.abs()).all())


def test_batches_without_rows(rt, scratch):
    vm = package()
    p = Paged(rt, [0, 0], [5, 0], pad=3)
    q = normal((3, 2, 64), "bf16", 1)
    o = torch.full_like(q, 4.0)
    for batch in (p.batch, vm.Batch(0, 0, 0, 0, 0, 3), vm.Batch(2, p.start.data_ptr(), p.length.data_ptr(), p.table.data_ptr(), p.table.shape[1], 0)):
        p.cache.Attend(batch, vm.Rows.Of(q), vm.Rows.Of(o), scratch, stream=_stream())
        p.cache.Write(batch, vm.Rows.Of(q), vm.Rows.Of(q), stream=_stream())
        p.cache.Read(batch, vm.Rows.Of(o), vm.Rows.Of(o), stream=_stream())
    assert p.cache.Status()["code"] == 0 and bool((o == 4.0).all())
    # a sequence without positions: its row attends to nothing, and the page list may be empty
    p = Paged(rt, [1], [0], lengths=[0])
    o = torch.full((1, 2, 64), 4.0, dtype=torch.bfloat16, device="cuda")
    p.cache.Attend(vm.Batch(1, p.start.data_ptr(), p.length.data_ptr(), 0, 0, 1), vm.Rows.Of(q[:1]), vm.Rows.Of(o), scratch, stream=_stream())
    assert p.cache.Status()["code"] == 0 and not bool(o.any())


@pytest.mark.parametrize("rows, q_heads", [(1, 2), (40, 8)])
def test_pages_and_batches_that_do_not_fit_are_reported(rt, scratch, rows, q_heads):
    """The kernels check what the host cannot see; the calls after the report are fine again."""
    vm = package()
    p = Paged(rt, [rows, rows, rows], [60, 60, 60], heads=2, q_heads=q_heads, page=16, spare=3)
    q = normal((p.n_rows, q_heads, 64), "bf16", 1)
    want, _, tol = p.attend(q, 0.125)
    tol = tol + half_step("bf16") * want.abs()

    def attend():
        o = torch.full_like(q, 4.0)
        p.cache.Attend(p.batch, vm.Rows.Of(q), vm.Rows.Of(o), scratch, stream=_stream())
        return o

    good = p.table.clone()
    for entry, number in ((0, -1), (3, p.n_pages), (1, 2 ** 31 - 1)):
        p.table[1, entry] = number
        o = attend()
        with pytest.raises(vm.InvalidArgument, match=f"sequence 1 names page {number} "):
            p.cache.Status()
        for b in (0, 2):
            s = slice(b * rows, (b + 1) * rows)
            assert bool(((o[s].double() - want[s]).abs() <= tol[s]).all())
        p.table.copy_(good)
    kv = normal((p.n_rows, 2, 64), "bf16", 2)
    p.table[2, (60 + rows - 1) // 16] = p.n_pages + 5
    before = [x.clone() for x in p.pages]
    p.cache.Write(p.batch, vm.Rows.Of(kv), vm.Rows.Of(kv), stream=_stream())
    with pytest.raises(vm.InvalidArgument, match="sequence 2 names page"):
        p.cache.Status()
    p.table.copy_(good)
    for i in range(2):
        p.pages[i].copy_(before[i])
    for what, tensor, at, value in (("length", p.length, 1, 10 ** 6), ("length", p.length, 1, -1), ("rows", p.start, 2, -3), ("rows", p.start, 3, 10 ** 6)):
        keep = tensor.clone()
        tensor[at] = value
        attend()
        with pytest.raises(vm.InvalidArgument, match="does not fit"):
            p.cache.Status()
        p.cache.Read(p.batch, vm.Rows.Of(kv), vm.Rows.Of(kv), stream=_stream())
        with pytest.raises(vm.InvalidArgument, match="does not fit"):
            p.cache.Status()
        tensor.copy_(keep)
    # more rows than max_rows said
    small = vm.Batch(3, p.start.data_ptr(), p.length.data_ptr(), p.table.data_ptr(), p.table.shape[1], p.n_rows, max(1, rows - 1))
    if rows > 1:
        o = torch.full_like(q, 4.0)
        p.cache.Attend(small, vm.Rows.Of(q), vm.Rows.Of(o), scratch, stream=_stream())
        with pytest.raises(vm.InvalidArgument, match="does not fit"):
            p.cache.Status()
        assert bool((o == 4.0).all())
    assert bool(((attend().double() - want).abs() <= tol).all()) and p.cache.Status()["code"] == 0


def test_a_cache_beyond_32_bits(rt, scratch):
    """Two pages 4.5 GB apart."""
    vm = package()
    stride = 2 ** 31 + 2 ** 28                                   # elements of 2 bytes
    room = torch.empty(stride + 4 * 16 * 2 * 64, dtype=torch.bfloat16, device="cuda")
    k, v = (room[i * 16 * 2 * 64:].as_strided((2, 16, 2, 64), (stride, 128, 64, 1)) for i in (0, 2))
    p = Paged(rt, [1, 20], [10, 5], heads=2, q_heads=2, page=16, spare=0)
    p.n_pages, p.pages = 2, [k, v]
    for i in range(2):
        p.pages[i].copy_(normal((2, 16, 2, 64), "bf16", i))
    p.rows, p.lengths = [20], [25]
    p.table = torch.tensor([[1, 0]], dtype=torch.int32, device="cuda")
    p.start, p.length = torch.tensor([0, 20], dtype=torch.int32, device="cuda"), torch.tensor([25], dtype=torch.int32, device="cuda")
    p.total = p.n_rows = p.max_rows = 20
    p.bind()
    kv = [normal((20, 2, 64), "bf16", 7 + i) for i in range(2)]
    p.cache.Write(p.batch, vm.Rows.Of(kv[0]), vm.Rows.Of(kv[1]), stream=_stream())
    out = [torch.empty_like(x) for x in kv]
    p.cache.Read(p.batch, vm.Rows.Of(out[0]), vm.Rows.Of(out[1]), stream=_stream())
    assert torch.equal(out[0], kv[0]) and torch.equal(out[1], kv[1])
    for rows in (20, 1):
        p.rows, p.n_rows, p.total, p.max_rows = [rows], rows, rows, rows
        p.start = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
        p.bind()
        q = normal((rows, 2, 64), "bf16", 3)
        o = torch.empty_like(q)
        p.cache.Attend(p.batch, vm.Rows.Of(q), vm.Rows.Of(o), scratch, stream=_stream())
        want, _, tol = p.attend(q, 0.125)
        assert bool(((o.double() - want).abs() <= tol + half_step("bf16") * want.abs()).all())
    assert p.cache.Status()["code"] == 0
