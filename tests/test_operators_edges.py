"""Attention over the paged cache where single values decide: scales far apart, NaN in one place, large scores, keys without a page.

Tolerances count as those of the other operator tests; rows of bf16 over 8-bit pages round their values to 16 bits beside the
weights, so there they are twice as wide (`_tol`)."""
from fractions import Fraction

import pytest

torch = pytest.importorskip("torch")

from conftest import package  # noqa: E402
from operator_refs import Paged, half_step, normal  # noqa: E402

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")


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


def _call(p, scratch, q, scale=None, **kw):
    o, lse = torch.full_like(q, 9.0), torch.full(q.shape[:2], 9.0, device="cuda")
    p.cache.Attend(p.batch, package().Rows.Of(q), package().Rows.Of(o), scratch, scale=scale, lse=lse.data_ptr(), stream=torch.cuda.current_stream().cuda_stream, **kw)
    return o, lse


def _tol(p, want, tol):
    return tol * (2 if p.dtype == "e4m3" and p.row_dtype == "bf16" else 1) + half_step(p.row_dtype) * want.abs()


def _near(got, want, tol):
    # (what is above a type's largest value, 65504 for f16, is an infinity in it)
    return bool((((got.double() - want).abs() <= tol) | (got == want.to(got.dtype)) & torch.isinf(got)).all())


def _place(p, b, pos):
    return int(p.table[b, pos // p.page]), pos % p.page


@pytest.mark.parametrize("dtype, row_dtype", [("bf16", "bf16"), ("f16", "f16"), ("e4m3", "bf16"), ("e4m3", "f16")])
@pytest.mark.parametrize("rows, past, q_heads, window", [(2, 0, 2, 0), (5, 40, 6, 7), (60, 0, 8, 0), (130, 300, 4, 50), (40, 3000, 8, 0)])
def test_a_nan_alone(rt, scratch, dtype, row_dtype, rows, past, q_heads, window):
    """One NaN in K, in V, in a scale of either, or in q, at the first key that a row sees: it shows wherever it is seen."""
    p = Paged(rt, [rows, 1], [past, 20], dtype=dtype, row_dtype=row_dtype, heads=2, q_heads=q_heads, dim=64, page=16, seed=5)
    clean_q = normal((p.n_rows, q_heads, 64), row_dtype, 8)
    want, want_lse, tol = p.attend(clean_q, 0.125, True, window)
    tol, lse_tol = _tol(p, want, tol), 2.0 ** -19 * (1 + want_lse.abs())
    clean = [x.clone() for x in p.pages], [None if s is None else s.clone() for s in p.scales]
    row = torch.arange(past, past + rows, device="cuda")
    head, group = 1, q_heads // 2
    mine = torch.zeros(p.n_rows, q_heads, dtype=torch.bool, device="cuda")
    for c in sorted({0, max(0, past - window + 1) if window else 0, past, past + 1}):
        sees = (c <= row) & ((c > row - window) if window else True)
        for what in ("k", "v", "q") + (("k scale", "v scale") if dtype == "e4m3" else ()):
            q = clean_q.clone()
            for i in range(2):
                p.pages[i].copy_(clean[0][i])
                if dtype == "e4m3":
                    p.scales[i].copy_(clean[1][i])
            mine[:] = False
            mine[:rows, head * group:(head + 1) * group] = sees[:, None]
            if what == "q":
                mine[:] = False
                mine[rows - 1, 1] = True
                q[rows - 1, 1, 63] = NAN
            elif what.endswith("scale"):
                p.scales["kv".index(what[0])][(*_place(p, 0, c), head)] = NAN
            elif dtype == "e4m3":
                p.pages["kv".index(what)].view(torch.uint8)[(*_place(p, 0, c), head, 17)] = 0x7F
            else:
                p.pages["kv".index(what)][(*_place(p, 0, c), head, 17)] = NAN
            o, lse = _call(p, scratch, q, window=window)
            assert p.cache.Status()["code"] == 0
            bad = mine[..., None].expand_as(o).clone()
            if what == "v":
                bad[..., :17] = bad[..., 18:] = False
            assert bool((torch.isnan(o) == bad).all()), (c, what)
            assert _near(o[~bad], want[~bad], tol[~bad]), (c, what)
            lse_bad = mine if what in ("k", "q", "k scale") else torch.zeros_like(mine)
            assert bool((torch.isnan(lse) == lse_bad).all()), (c, what)
            assert _near(lse[~lse_bad], want_lse[~lse_bad], lse_tol[~lse_bad]), (c, what)


# rows, past, heads, q heads, row type: parts of a tile's keys by several CTAs, whole tiles, single tokens
FAR = [(20, 6000, 1, 8, "bf16"), (20, 6000, 1, 8, "f16"), (130, 3, 2, 4, "bf16"), (130, 3, 2, 4, "f16"), (300, 2001, 16, 16, "bf16"), (2, 701, 2, 8, "bf16"), (2, 701, 2, 8, "f16")]


@pytest.mark.parametrize("far", [2.0 ** 9, 2.0 ** 13, 2.0 ** 20])
@pytest.mark.parametrize("causal, window", [(True, 0), (False, 0), (True, 37)])
@pytest.mark.parametrize("rows, past, heads, q_heads, row_dtype", FAR)
def test_scales_far_apart(rt, scratch, rows, past, heads, q_heads, row_dtype, causal, window, far):
    """Neighbours whose V scales are `far` apart, at the end of a sequence that ends inside a block, and where rows begin and end to see."""
    p = Paged(rt, [rows, 3], [past, 50], dtype="e4m3", row_dtype=row_dtype, heads=heads, q_heads=q_heads, dim=64, seed=3)
    length = rows + past
    for pos in range(length - 9, length, 2):
        p.scales[1][_place(p, 0, pos)] /= far
    for pos in (past, past + 1, max(0, past - 30)):
        p.scales[1][_place(p, 0, pos)] *= far
    q = normal((p.n_rows, q_heads, 64), row_dtype, 8, 2.0)
    want, want_lse, tol = p.attend(q, 0.125, causal, window)
    o, lse = _call(p, scratch, q, causal=causal, window=window)
    assert p.cache.Status()["code"] == 0
    assert _near(o, want, _tol(p, want, tol))
    assert _near(lse, want_lse, 2.0 ** -19 * (1 + want_lse.abs()))


@pytest.mark.parametrize("dtype, row_dtype", [("bf16", "bf16"), ("f16", "f16"), ("e4m3", "bf16"), ("e4m3", "f16")])
def test_rows_worked_out_again_behind_the_products(rt, scratch, dtype, row_dtype):
    """Whole tiles and parts of them, all of whose rows see a V that is not finite: the batch's other tiles are done as ever, captured too, and
    the call after finds nothing of it."""
    rows, past = [70] * 40 + [300], list(range(0, 800, 20)) + [9000]
    p = Paged(rt, rows, past, dtype=dtype, row_dtype=row_dtype, heads=4, q_heads=16, dim=64, page=48, seed=5)
    q = normal((p.n_rows, 16, 64), row_dtype, 8)
    want, want_lse, tol = p.attend(q, 0.125)
    tol = _tol(p, want, tol)
    clean, _ = _call(p, scratch, q)
    assert _near(clean, want, tol)
    keep = p.pages[1].clone()
    bad = torch.zeros_like(q, dtype=torch.bool)
    for b in (0, 3, 17, 40):                                     # a NaN at the first key, value 9 of cache head 2; another at the last
        for pos, d in ((0, 9), (p.lengths[b] - 1, 11)):
            at = (*_place(p, b, pos), 2, d)
            if dtype == "e4m3":
                p.pages[1].view(torch.uint8)[at] = 0x7F
            else:
                p.pages[1][at] = NAN
        first = sum(rows[:b])
        bad[first:first + rows[b], 8:12, 9] = True
        bad[first + rows[b] - 1, 8:12, 11] = True
    o, lse = torch.empty_like(q), torch.empty(q.shape[:2], device="cuda")
    r = package().Rows.Of
    side, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=side):
        p.cache.Attend(p.batch, r(q), r(o), scratch, lse=lse.data_ptr(), stream=side.cuda_stream)
    for turn in range(2):
        o.fill_(9.0)
        g.replay()
        torch.cuda.synchronize()
        assert p.cache.Status()["code"] == 0
        assert bool((torch.isnan(o) == bad).all()) and _near(o[~bad], want[~bad], tol[~bad])
        assert _near(lse, want_lse, 2.0 ** -19 * (1 + want_lse.abs()))
    p.pages[1].copy_(keep)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(o, clean)


@pytest.mark.parametrize("dtype, row_dtype", [("f16", "f16"), ("bf16", "bf16"), ("e4m3", "bf16"), ("e4m3", "f16")])
@pytest.mark.parametrize("rows, past, q_heads", [(1, 300, 4), (3, 40, 8), (40, 100, 4), (300, 0, 2), (33, 5000, 2)])
@pytest.mark.parametrize("base", [1250.0, -1250.0, 2048.0, 3000.0, -3000.0, 4096.0, -4160.0])
def test_large_scores(rt, scratch, dtype, row_dtype, rows, past, q_heads, base):
    """Scores around `base` that differ by a few: what is common to a row's scores cancels, however large it is."""
    p = Paged(rt, [rows], [past], dtype=dtype, row_dtype=row_dtype, heads=1, q_heads=q_heads, dim=64, page=16, seed=6)
    if dtype == "e4m3":                                          # (codes 256 and a scale of 2^-3: 32 exactly)
        p.pages[0].view(torch.uint8)[..., 0] = 0x78
        p.scales[0].fill_(2.0 ** -3)
        p.pages[0].view(torch.uint8)[..., 1:] = torch.randint(0x28, 0x38, p.pages[0][..., 1:].shape, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda", dtype=torch.uint8)
    else:
        p.pages[0][..., 0] = 32.0
    q = normal((rows, q_heads, 64), row_dtype, 8, 0.25)
    q[..., 0] = base / 32.0                                      # (at most 7 bits: exact)
    want, want_lse, tol = p.attend(q, 1.0)
    o, lse = _call(p, scratch, q, scale=1.0)
    assert p.cache.Status()["code"] == 0
    assert _near(o, want, _tol(p, want, tol))
    # a score and its sum in f32: 64 terms, all but a few of them small beside the first
    assert _near(lse, want_lse, 16 * 2.0 ** -24 * want_lse.abs() + 2.0 ** -17)


def _without(p, b, q, scale, absent, window=0):
    """Sequence b's rows in 64 bits, keys of `absent` left out: out, lse, sum w |v|, the largest sum |q k|."""
    n, length, g = p.rows[b], p.lengths[b], p.q_heads // p.heads
    first = sum(p.rows[:b])
    k, v = (p.values(b, i).repeat_interleave(g, 1).transpose(0, 1) for i in (0, 1))
    x = q[first:first + n].double().transpose(0, 1)
    row, key = torch.arange(length - n, length, device="cuda")[:, None], torch.arange(length, device="cuda")[None]
    seen = (key <= row) & ~absent[None]
    if window:
        seen = seen & (key > row - window)
    s = (x @ k.transpose(1, 2) * scale).masked_fill(~seen, -INF)
    lse = torch.logsumexp(s, -1)
    w = torch.where(seen, torch.exp(s - lse[..., None]), torch.zeros_like(s))
    reach = (x.abs() @ k.abs().transpose(1, 2) * scale).amax(-1)
    return [t.transpose(0, 1) for t in (w @ v, lse, w @ v.abs(), reach)]


@pytest.mark.parametrize("dtype, row_dtype", [("bf16", "bf16"), ("f16", "f16"), ("e4m3", "bf16"), ("e4m3", "f16")])
@pytest.mark.parametrize("rows, past, q_heads, page, window", [(1, 200, 4, 16, 0), (3, 60, 8, 7, 0), (2, 500, 2, 64, 90), (40, 100, 4, 16, 0), (150, 4000, 4, 24, 0), (300, 37, 2, 5, 60)])
def test_keys_without_a_page_are_absent(rt, scratch, dtype, row_dtype, rows, past, q_heads, page, window):
    """The sequence that names pages outside the cache: its rows over the keys that there are."""
    p = Paged(rt, [2, rows], [9, past], dtype=dtype, row_dtype=row_dtype, heads=2, q_heads=q_heads, dim=64, page=page, seed=7)
    q = (normal((p.n_rows, q_heads, 64), row_dtype, 8).abs() + 0.25).to(normal((1,), row_dtype, 0).dtype)
    if dtype == "e4m3":
        p.pages[0].view(torch.uint8).bitwise_or_(0x80)           # scores below 0: a key of zeros would outweigh all others
    else:
        p.pages[0].copy_(-p.pages[0].abs())
    length = rows + past
    last = (length - 1) // page
    for entries in ((0,), (last,), (last // 2, last // 2 + 1), tuple(range(0, last + 1, 2)), tuple(range(last + 1))):
        absent = torch.zeros(length, dtype=torch.bool, device="cuda")
        for e in entries:
            absent[e * page:(e + 1) * page] = True
        want, want_lse, size, reach = _without(p, 1, q, 0.125, absent, window)
        keep = p.table.clone()
        for i, e in enumerate(entries):
            p.table[1, e] = -1 if i % 2 else p.n_pages
        o, lse = _call(p, scratch, q, window=window)
        if bool(absent[max(0, past + 1 - window) if window else 0:].any()):       # (what nobody sees is not looked up)
            with pytest.raises(package().InvalidArgument, match="sequence 1 names page"):
                p.cache.Status()
        assert p.cache.Status()["code"] == 0
        p.table.copy_(keep)
        got, got_lse = o[2:], lse[2:]
        none = want_lse == -INF
        assert bool((got_lse[none] == -INF).all()) and not bool(got[none].any())
        off = (2 * (68 * 2.0 ** -24 * reach + 2.0 ** -22 + (length / 8 + 16) * 2.0 ** -24) + 2 * half_step("f16" if dtype == "e4m3" else row_dtype))[..., None]
        assert _near(got[~none], want[~none], (off * size + half_step(row_dtype) * want.abs())[~none]), entries
        assert _near(got_lse[~none], want_lse[~none], (2 * 68 * 2.0 ** -24 * reach + 2.0 ** -19 * (1 + want_lse.abs()))[~none]), entries


@pytest.mark.parametrize("rows", [1, 4, 50])
def test_queries_of_any_size_over_8_bit_pages(rt, scratch, rows):
    """Rows of bf16 between 2^-60 and 2^126, K's scales the other way round."""
    p = Paged(rt, [rows], [70], dtype="e4m3", heads=2, q_heads=4, dim=64, page=16, seed=4)
    scales, base = p.scales[0].clone(), normal((rows, 4, 64), "bf16", 8)
    for e in (-60, 0, 90, 113, 115, 120, 123):
        q = (base.double() * 2.0 ** e).bfloat16()
        p.scales[0].copy_(scales * 2.0 ** -e)
        want, want_lse, tol = p.attend(q, 0.125)
        o, lse = _call(p, scratch, q)
        assert p.cache.Status()["code"] == 0
        assert _near(o, want, _tol(p, want, tol)), e
        assert _near(lse, want_lse, 2.0 ** -19 * (1 + want_lse.abs())), e


@pytest.mark.parametrize("dtype, row_dtype, dim", [("bf16", "bf16", 128), ("f16", "f16", 64), ("e4m3", "bf16", 128), ("e4m3", "f16", 64)])
def test_waits_that_run_out_are_reported(rt, scratch, dtype, row_dtype, dim):
    """With no time for any wait the roles of a CTA give up one after another, wherever they are: each call ends, and says so; those after it are
    as ever."""
    vm = package()
    p = Paged(rt, [300, 40], [2000, 100], dtype=dtype, row_dtype=row_dtype, heads=4, q_heads=8, dim=dim, page=16, seed=2)
    q = normal((p.n_rows, 8, dim), row_dtype, 8)
    clean, _ = _call(p, scratch, q)
    want, _, tol = p.attend(q, dim ** -0.5)
    assert _near(clean, want, _tol(p, want, tol)) and p.cache.Status()["code"] == 0
    reported = 0
    for turn in range(12):
        p.cache.set_wait_budget_ns(turn // 4 * 1000)             # (0: the first look has to do)
        o, _ = _call(p, scratch, q)
        try:
            assert p.cache.Status()["code"] == 0 and torch.equal(o, clean)
        except vm.DeadlineExceeded as e:
            assert "tensor cores" in str(e)
            reported += 1
    assert reported > 0
    p.cache.set_wait_budget_ns(2_000_000_000)
    for _ in range(2):
        assert torch.equal(_call(p, scratch, q)[0], clean) and p.cache.Status()["code"] == 0


def test_handles_are_made_while_the_device_is_busy(rt, scratch):
    """A server makes and captures for a new batch while its last one runs: nothing of that is waited for."""
    vm = package()
    p = Paged(rt, [3], [20], heads=2, dim=64)
    vm.Rope.Create(rt, 64, 2, 2, "bf16")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    ends = []
    for stream in (torch.cuda.current_stream(), side):
        with torch.cuda.stream(stream):
            torch.cuda._sleep(2_000_000_000)                     # about a second
            ends.append(torch.cuda.Event())
            ends[-1].record()
    first = p.cache                                              # (a handle that goes waits: its memory may be in use)
    p.bind()
    rope, other = vm.Rope.Create(rt, 64, 2, 2, "bf16"), vm.Scratch.Create(rt)
    assert not any(e.query() for e in ends)
    torch.cuda.synchronize()
    q = normal((3, 2, 64), "bf16", 1)
    want, _, tol = p.attend(q, 0.125)
    assert _near(_call(p, other, q)[0], want, _tol(p, want, tol)) and p.cache.Status()["code"] == 0
    out, pos = torch.empty_like(q), torch.zeros(3, dtype=torch.int32, device="cuda")
    r = vm.Rows.Of
    rope.Apply(3, pos.data_ptr(), r(q), r(q), r(out), r(torch.empty_like(q)))
    assert torch.equal(out, q)                                   # (position 0)
    first.close()


def test_handles_that_go_during_a_capture(rt, scratch):
    """As a collector does it: the capture is not ended by it, and its graph runs."""
    vm = package()
    p = Paged(rt, [3], [20], heads=2, dim=64)
    gone = [vm.Rope.Create(rt, 64, 2, 2, "bf16"), vm.Scratch.Create(rt), p.cache]
    p.bind()
    q = normal((3, 2, 64), "bf16", 1)
    want, _ = _call(p, scratch, q)
    o, r = torch.zeros_like(q), vm.Rows.Of
    side, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=side):
        for handle in gone:
            handle.close()
        p.cache.Attend(p.batch, r(q), r(o), scratch, stream=side.cuda_stream)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(o, want) and p.cache.Status()["code"] == 0


def test_results_over_inputs_or_themselves_are_refused(rt, scratch):
    vm = package()
    p = Paged(rt, [2, 3], [20, 5], heads=2, q_heads=4, dim=64)
    r = vm.Rows.Of
    flat = normal((6 * 8 * 64,), "bf16", 1)
    fused = flat[:5 * 8 * 64].view(5, 8, 64)
    q, beside = fused[:, :4], fused[:, 4:]
    for out in (q, flat[64:64 + 5 * 512].view(5, 8, 64)[:, :4], flat[512:512 + 5 * 512].view(5, 8, 64)[:, :4], fused[:, 1:5], fused[:, 3:7], flat[1:1 + 5 * 512].view(5, 8, 64)[:, :4],
                flat[512 - 63:512 - 63 + 5 * 512].view(5, 8, 64)[:, :4], flat[256:256 + 5 * 256].view(5, 4, 64)):
        with pytest.raises(vm.InvalidArgument, match="over q"):
            p.cache.Attend(p.batch, r(q), r(out), scratch)
    for out in (beside, flat.new_empty(5, 4, 64), fused.new_empty(4, 5, 64).transpose(0, 1)):
        p.cache.Attend(p.batch, r(q), r(out), scratch)
    for out in (fused.new_empty(1, 4, 64).expand(5, 4, 64), fused.new_empty(5, 1, 64).expand(5, 4, 64), fused.new_empty(2000).as_strided((5, 4, 64), (128, 64, 1)),
                fused.new_empty(2000).as_strided((5, 4, 64), (63, 400, 1))):
        with pytest.raises(vm.InvalidArgument, match="over each other"):
            p.cache.Attend(p.batch, r(q), r(out), scratch)
    for out in (fused.new_empty(1, 2, 64).expand(5, 2, 64), fused.new_empty(5, 1, 64).expand(5, 2, 64)):
        with pytest.raises(vm.InvalidArgument, match="over each other"):
            p.cache.Read(p.batch, r(q[:, :2].clone()), r(out))
    p.cache.Attend(p.batch, r(q), r(fused.new_empty(2000).as_strided((5, 4, 64), (65, 390, 1))), scratch)      # (heads first, a gap in each row)
    pos = torch.arange(5, dtype=torch.int32, device="cuda")
    k, other = fused[:, 4:6], fused.new_empty(5, 4, 64)
    rope = vm.Rope.Create(rt, 64, 4, 2, "bf16")
    want = [torch.empty_like(t) for t in (q, k)]
    rope.Apply(5, pos.data_ptr(), r(q), r(k), r(want[0]), r(want[1]))
    for q_out, k_out, part in ((fused[:, 1:5], k, "over q"), (q, fused[:, 3:5], "over q"), (k.new_empty(5, 4, 64), fused[:, 5:7], "over k"), (fused[:, 2:6], k.new_empty(5, 2, 64), "over q"),
                               (other, other[:, :2], "other result"), (other[:1].expand(5, 4, 64), k, "over each other")):
        with pytest.raises(vm.InvalidArgument, match=part):
            rope.Apply(5, pos.data_ptr(), r(q), r(k), r(q_out), r(k_out))
    g = [normal(t.shape, "bf16", 5) for t in (q, k)]
    with pytest.raises(vm.InvalidArgument, match="over gradient of a result"):
        rope.ApplyBackward(5, pos.data_ptr(), None, None, r(g[0]), r(g[1]), r(other), r(g[0][:, 2:]))
    rope.Apply(5, pos.data_ptr(), r(q), r(k), r(q), r(k))        # over its own inputs, in the fused rows
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    one = vm.Rope.Create(rt, 64, 1, 1, "bf16")                   # one row, one head: strides say nothing
    x = normal((3, 64), "bf16", 1)
    one.Apply(1, pos.data_ptr(), vm.Rows(x[0].data_ptr(), "bf16", (1, 1, 64), (0, 0)), vm.Rows(x[1].data_ptr(), "bf16", (1, 1, 64), (7, 3)), vm.Rows(x[0].data_ptr(), "bf16", (1, 1, 64), (1, 1)),
              vm.Rows(x[2].data_ptr(), "bf16", (1, 1, 64)))
    assert torch.equal(x[2], x[1]) and p.cache.Status()["code"] == 0


def _sine_and_cosine(position, frequency):
    """To 2^-80 or so: the angle as a fraction, pi to 60 digits, series."""
    pi = Fraction(3141592653589793238462643383279502884197169399375105820974944, 10 ** 60)
    angle = (position * Fraction(frequency)) % (2 * pi)
    angle = Fraction(round(angle * 2 ** 120), 2 ** 120)
    out = []
    for term, k in ((angle, 1), (Fraction(1), 0)):
        total = Fraction(0)
        while abs(term) > Fraction(1, 2 ** 90):
            total += term
            k += 2
            term = Fraction(round(-term * angle * angle / (k * (k - 1)) * 2 ** 120), 2 ** 120)
        out.append(float(total))
    return out


def test_sines_of_far_positions(rt):
    """Rows of pairs (1, 0) in f32 come back as cosine and sine."""
    vm = package()
    freq = [1.0, 0.5 ** 0.5, 10000.0 ** -0.25, 1e-2, 1.0 - 2.0 ** -53, 3e-4, 1e-4, 2.0 ** -20]
    pos = [0, 1, 17, 131071, 999999, 2 ** 24 + 1, 2 ** 27 - 1, -(2 ** 27) + 3, 2 ** 30 + 12345, 2 ** 31 - 1, -(2 ** 31), 1686629713 // 5]
    rope = vm.Rope.Create(rt, 16, 1, 0, "f32", frequencies=freq)
    x = torch.zeros(len(pos), 1, 16, device="cuda")
    x[..., :8] = 1.0
    out = torch.empty_like(x)
    rope.Apply(len(pos), torch.tensor(pos, dtype=torch.int32, device="cuda"), vm.Rows.Of(x), None, vm.Rows.Of(out), None, stream=torch.cuda.current_stream().cuda_stream)
    for i, p in enumerate(pos):
        for j, f in enumerate(freq):
            sine, cosine = _sine_and_cosine(p, f)
            off = max(abs(float(out[i, 0, j]) - cosine), abs(float(out[i, 0, 8 + j]) - sine))
            assert off <= (2.0 ** -22 if abs(p) * f < 2 ** 27 else 2.0 ** -20), (p, f, off * 2 ** 24)


@pytest.mark.parametrize("row_dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rows, q_heads", [(1, 4), (4, 8), (40, 4), (200, 2)])
@pytest.mark.parametrize("apart, other", [(2.0 ** 19, 32), (2.0 ** 14, 1)])
def test_a_small_v_scale_under_all_the_weight(rt, scratch, row_dtype, rows, q_heads, apart, other):
    """A key that has the weight counts in full beside one that has none and a V scale `apart` times larger."""
    p = Paged(rt, [rows], [100], dtype="e4m3", row_dtype=row_dtype, heads=2, q_heads=q_heads, dim=64, page=16, seed=6)
    c = 35
    p.pages[0].view(torch.uint8)[...] = 0x30                     # scores alike, but for key c's
    p.pages[0].view(torch.uint8)[_place(p, 0, c)] = 0x50
    p.scales[0].fill_(1.0)
    p.scales[1].fill_(1.0 / 448)
    p.scales[1][_place(p, 0, c + other)] *= apart
    q = torch.full((rows, q_heads, 64), 1.0, device="cuda").to(normal((1,), row_dtype, 0).dtype)
    want, want_lse, tol = p.attend(q, 0.125)                     # (8 x (16 - 0.5) = 60 and more between them: e^-60 x 2^19 is nothing)
    assert _near(want, p.values(0, 1)[c].repeat_interleave(q_heads // 2, 0).expand_as(want), 2.0 ** -40)
    o, lse = _call(p, scratch, q)
    assert p.cache.Status()["code"] == 0
    # values below f16's smallest normal one are off by half of its smallest step, 2^-25: of V, which is held 2^7 higher, over a power above its 16 keys' scales
    low = 2.0 ** -32 * 2 * float(p.scales[1].max()) if other == 1 else 0.0
    assert _near(o, want, _tol(p, want, tol) + low) and _near(lse, want_lse, 2.0 ** -19 * (1 + want_lse.abs()))
