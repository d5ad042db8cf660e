"""The operators beside the programs as a serving loop has them: on streams, captured and replayed while the batch changes, sharing a
scratch in order and having one each at once, from two threads, and between loaded programs' products."""
import threading

import pytest

torch = pytest.importorskip("torch")

from conftest import package  # noqa: E402
from operator_refs import U, Paged, half_step, normal, rope  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rt():
    r = package().Runtime.Create(0)
    yield r
    r.close()


class Layer:
    """One layer's rope, cache and rows for a batch; `step` makes its calls on a stream."""

    def __init__(self, rt, rows, past, *, seed, max_rows=None, q_heads=4, dtype="bf16", pad=0, **kw):
        vm = package()
        self.p = Paged(rt, rows, past, heads=2, q_heads=q_heads, dim=64, page=16, dtype=dtype, seed=seed, max_rows=max_rows, pad=pad, **kw)
        n, hq = self.p.n_rows, q_heads
        self.freq = vm.RopeFrequencies(64)
        self.rope = vm.Rope.Create(rt, 64, hq, 2, "bf16", frequencies=self.freq, norm=True, eps=1e-6)
        self.scratch = vm.Scratch.Create(rt)
        self.qkv = normal((n, hq + 4, 64), "bf16", seed + 3, 2.0)
        self.weight = (1.0 + 0.2 * normal((2, 64), "f32", seed + 4))
        self.q, self.k = torch.empty((n, hq, 64), dtype=torch.bfloat16, device="cuda"), torch.empty((n, 2, 64), dtype=torch.bfloat16, device="cuda")
        self.out, self.lse = torch.zeros_like(self.q), torch.zeros((n, hq), device="cuda")
        self.pos = torch.zeros(n, dtype=torch.int32, device="cuda")
        self.hq = hq
        self.place()
        r = vm.Rows.Of
        self.views = [r(self.qkv[:, :hq]), r(self.qkv[:, hq:hq + 2]), r(self.qkv[:, hq + 2:]), r(self.q), r(self.k), r(self.out)]

    def place(self):
        """Positions of the rows, by the batch as it is."""
        start, length = self.p.start.cpu().tolist(), self.p.length.cpu().tolist()
        at = [x for b, n in enumerate(length) for x in range(n - (start[b + 1] - start[b]), n)]
        self.pos[:len(at)] = torch.tensor(at, dtype=torch.int32, device="cuda")

    def step(self, stream, scratch=None):
        q, k, v, q_out, k_out, out = self.views
        p = self.p
        self.rope.Apply(p.n_rows, self.pos.data_ptr(), q, k, q_out, k_out, self.weight[0].data_ptr(), self.weight[1].data_ptr(), stream=stream)
        p.cache.Write(p.batch, k_out, v, stream=stream)
        p.cache.Attend(p.batch, q_out, out, scratch or self.scratch, lse=self.lse.data_ptr(), stream=stream)

    def fine(self):
        """The attention's results for the queries and the pages as they are now."""
        assert self.p.cache.Status()["code"] == 0
        want, lse, tol = self.p.attend(self.q, 0.125)
        n = want.shape[0]
        assert bool(((self.out[:n].double() - want).abs() <= tol + half_step("bf16") * want.abs()).all())
        # a score: 64 terms of at most sum |q k| <= |q| |k|; the logarithm and the sum a few roundings
        size = self.q.double().norm(dim=-1).amax() * max(float(self.p.values(b, 0).norm(dim=-1).amax()) for b in range(len(self.p.rows))) * 0.125
        assert bool(((self.lse[:n].double() - lse).abs() <= 2 * (68 * U * size + 2.0 ** -20) * (1 + lse.abs())).all())

    def results(self):
        return [t.clone() for t in (self.q, self.k, self.out, self.lse, *self.p.pages)]


SHAPES = [([1, 1, 1], [70, 3, 500], 4, "bf16"), ([40, 1, 129], [10, 33, 200], 4, "bf16"), ([1, 60], [100, 0], 8, "e4m3")]


@pytest.mark.parametrize("rows, past, q_heads, dtype", SHAPES)
def test_in_the_order_of_the_stream_they_are_given(rt, rows, past, q_heads, dtype):
    layer = Layer(rt, rows, past, seed=5, q_heads=q_heads, dtype=dtype)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)                     # about 10 ms: what comes next is queued behind it
        layer.qkv.mul_(0.5)
        layer.step(side.cuda_stream)
        out = layer.out * 1.0
    side.synchronize()
    assert torch.equal(out, layer.out) and bool(out.any())
    freq = layer.freq
    x = layer.qkv[:, :layer.hq].double()
    want = rope(x, layer.weight[0].double(), layer.pos, freq, 64, False, True, 1e-6, 1.0)
    reach = 2 * x.abs().amax(-1, keepdim=True) * torch.rsqrt((x * x).mean(-1, keepdim=True)) * layer.weight[0].abs().max()
    assert bool(((layer.q.double() - want).abs() <= half_step("bf16") * want.abs() + 60 * U * reach).all())
    layer.fine()
    before = layer.results()
    layer.step(0)                                         # the default stream, the same once more
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(before, layer.results()))


@pytest.mark.parametrize("rows, past, q_heads, dtype", SHAPES)
def test_captured_and_replayed_while_the_batch_changes(rt, rows, past, q_heads, dtype):
    """Lengths, rows, pages and positions are read when a graph runs; rows behind the last sequence stay as they are."""
    layer = Layer(rt, rows, past, seed=6, q_heads=q_heads, dtype=dtype, pad=3, extra_pages=30, spare=60)
    p = layer.p
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        layer.step(side.cuda_stream)
    used = set(p.table[p.table >= 0].cpu().tolist())
    free = [x for x in range(p.n_pages) if x not in used]
    for turn in range(3):
        layer.out.fill_(5.0)
        g.replay()
        torch.cuda.synchronize()
        layer.fine()
        assert bool((layer.out[p.total:] == 5.0).all())
        # every sequence grows by what it has been given, the last one has a row less each time
        for b in range(len(p.rows)):
            p.lengths[b] += p.rows[b]
            need = -(-p.lengths[b] // p.page)
            for e in range(p.table.shape[1]):
                if e < need and int(p.table[b, e]) < 0:
                    p.table[b, e] = free.pop()
        if p.rows[-1] > 1:
            p.rows[-1] -= 1
            p.lengths[-1] -= 1
            p.total -= 1
            p.start[-1] -= 1
        p.length.copy_(torch.tensor(p.lengths, dtype=torch.int32))
        assert max(-(-n // p.page) for n in p.lengths) <= p.table.shape[1]
        layer.place()
        layer.qkv.copy_(normal(layer.qkv.shape, "bf16", 50 + turn, 2.0))


def test_two_graphs_with_one_scratch_and_two_streams_with_one_each(rt):
    a, b = Layer(rt, *SHAPES[1][:2], seed=11), Layer(rt, [1] * 20, list(range(100, 2100, 100)), seed=12)
    wants = []
    for layer in (a, b):
        layer.step(0)
        torch.cuda.synchronize()
        layer.fine()
        wants.append(layer.results())
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    graphs = []
    for layer in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            for _ in range(3):
                layer.step(side.cuda_stream, a.scratch)
        graphs.append(g)
    for layer in (a, b):
        layer.out.zero_()
    with torch.cuda.stream(side):
        for i in range(6):
            graphs[i % 2].replay()
    torch.cuda.synchronize()
    for layer, want in zip((a, b), wants):
        assert all(torch.equal(x, y) for x, y in zip(want, layer.results()))
        layer.out.zero_()
    torch.cuda.synchronize()
    for _ in range(10):                                   # (at once, each with its own)
        a.step(side.cuda_stream)
        b.step(other.cuda_stream)
    torch.cuda.synchronize()
    for layer, want in zip((a, b), wants):
        assert all(torch.equal(x, y) for x, y in zip(want, layer.results()))


def test_from_two_threads(rt):
    layers = [Layer(rt, *SHAPES[i][:2], seed=20 + i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in layers]
    torch.cuda.synchronize()
    errors = []

    def work(layer, stream):
        try:
            for _ in range(50):
                layer.step(stream.cuda_stream)
                with pytest.raises(package().InvalidArgument, match="window"):
                    layer.p.cache.Attend(layer.p.batch, layer.views[3], layer.views[5], layer.scratch, causal=False, window=4)
        except BaseException as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=x) for x in zip(layers, streams)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    torch.cuda.synchronize()
    for layer in layers:
        layer.fine()


def test_gradients_captured_and_replayed(rt):
    """Rotary positions' gradients in a graph: the same bits as called, with the inputs of the time of the replay."""
    vm = package()
    n, hq, hk = 700, 5, 2
    handle, scratch = vm.Rope.Create(rt, 96, hq, hk, "bf16", rot_dim=64, norm=True), vm.Scratch.Create(rt)
    x, dy = ([normal((n, h, 96), "bf16", s + i) for i, h in enumerate((hq, hk))] for s in (1, 3))
    w = 1.0 + 0.1 * normal((2, 96), "f32", 9)
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    dx, dw = [torch.empty_like(t) for t in x], torch.empty((2, 96), device="cuda")
    r = vm.Rows.Of

    def back(stream):
        handle.ApplyBackward(n, pos.data_ptr(), r(x[0]), r(x[1]), r(dy[0]), r(dy[1]), r(dx[0]), r(dx[1]), w[0].data_ptr(), w[1].data_ptr(), dw[0].data_ptr(),
                             dw[1].data_ptr(), scratch, stream=stream)

    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        back(side.cuda_stream)
    for turn in range(2):
        back(0)
        want = [t.clone() for t in (*dx, dw)]
        for t in (*dx, dw):
            t.fill_(3.0)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, (*dx, dw)))
        pos.add_(5)
        dy[0].neg_()


def test_refused_calls_leave_everything(rt):
    vm = package()
    layer = Layer(rt, [1, 1], [20, 30], seed=40)
    p, r, scratch = layer.p, vm.Rows.Of, layer.scratch
    q, k, v, q_out, k_out, out = layer.views
    layer.step(0)
    torch.cuda.synchronize()
    before = layer.results()
    f32 = torch.zeros((2, 2, 64), device="cuda")
    bad = [
        (lambda: p.cache.Attend(p.batch, q_out, out, None), "null scratch"),
        (lambda: p.cache.Attend(p.batch, q_out, q_out, scratch), "over q"),
        (lambda: p.cache.Attend(p.batch, q_out, None, scratch), "out: missing"),
        (lambda: p.cache.Attend(p.batch, k_out, out, scratch), "q: bf16"),
        (lambda: p.cache.Attend(p.batch, q_out, out, scratch, scale=float("nan")), "scale"),
        (lambda: p.cache.Attend(p.batch, q_out, out, scratch, causal=False, window=3), "needs causal"),
        (lambda: p.cache.Attend(p.batch, q_out, out, scratch, window=-1), "window"),
        (lambda: p.cache.Attend(p.batch, q_out, out, scratch, lse=layer.lse.data_ptr() + 2), "lse"),
        (lambda: p.cache.Attend(vm.Batch(2, p.start.data_ptr(), p.length.data_ptr(), p.table.data_ptr(), p.table.shape[1], 3), q_out, out, scratch), "3 or more"),
        (lambda: p.cache.Attend(vm.Batch(2, p.start.data_ptr(), 0, p.table.data_ptr(), p.table.shape[1], 2), q_out, out, scratch), "null row_start"),
        (lambda: p.cache.Attend(vm.Batch(2, p.start.data_ptr(), p.length.data_ptr(), p.table.data_ptr(), p.table.shape[1], 2, pages_stride=1), q_out, out, scratch), "pages_stride"),
        (lambda: p.cache.Write(p.batch, q_out, v), "k: bf16"),
        (lambda: p.cache.Write(p.batch, k_out, r(f32)), "v: f32"),
        (lambda: p.cache.Read(p.batch, k_out, None), "v: missing"),
        (lambda: r(f32.cpu()), "device memory"),
        (lambda: r(f32.transpose(1, 2)), "stride 1"),
        (lambda: r(f32[0]), r"\[rows, heads, head_dim\]"),
        (lambda: r(f32.double()), "rows of type"),
        (lambda: vm.Rows(f32.data_ptr() + 1, "f32", (2, 2, 64)) and layer.rope.Apply(2, layer.pos.data_ptr(), vm.Rows(layer.q.data_ptr() + 1, "bf16", (2, 4, 64)), k, q_out, k_out), "not aligned"),
        (lambda: layer.rope.Apply(2, 0, q, k, q_out, k_out), "null positions"),
        (lambda: layer.rope.Apply(2, layer.pos.data_ptr() + 1, q, k, q_out, k_out), "positions"),
        (lambda: layer.rope.Apply(3, layer.pos.data_ptr(), q, k, q_out, k_out), "3 or more"),
        (lambda: layer.rope.Apply(2, layer.pos.data_ptr(), q, k, q_out, q_out), "k_out: bf16"),
        (lambda: layer.rope.ApplyBackward(2, layer.pos.data_ptr(), q, k, q_out, k_out, q_out, k_out, dq_weight=f32.data_ptr()), "need a scratch"),
        (lambda: layer.rope.ApplyBackward(2, layer.pos.data_ptr(), None, k, q_out, k_out, q_out, k_out), "q: missing"),
    ]
    for call, part in bad:
        with pytest.raises(vm.InvalidArgument, match=part):
            call()
    rows32 = Paged(rt, [1], [3], dtype="bf16", row_dtype="f32", heads=2, dim=64)
    with pytest.raises(Exception, match="f32 rows"):
        rows32.cache.Attend(rows32.batch, vm.Rows.Of(f32), vm.Rows.Of(torch.empty_like(f32)), scratch)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(before, layer.results())) and p.cache.Status()["code"] == 0


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
def test_a_decoder_layer_between_loaded_products(rt, cache):
    """Prompts of different lengths, then tokens one by one: a program's product makes queries, keys and values, the operators take them
    from there as views, and another product reads the attention's rows. Each part against its formula on what it was given."""
    import plan_programs as progs
    vm = package()
    width, hq, hk, dim = 256, 4, 2, 64
    prompts, steps = [37, 1, 90], 3
    total = sum(prompts)
    wide = (hq + 2 * hk) * dim
    x0 = normal((total + steps * len(prompts), width), "bf16", 1)
    w_in, w_out = normal((width, wide), "bf16", 2, width ** -0.5), normal((hq * dim, width), "bf16", 3, (hq * dim) ** -0.5)
    programs = {n: [vm.LoadedProgram.Load(rt, vm.VmProgram.Parse(progs.products("bf16", mkn).blob())) for mkn in ((n, width, wide), (n, hq * dim, width))]
                for n in (total, len(prompts))}
    p = Paged(rt, prompts, [0] * len(prompts), dtype=cache, heads=hk, q_heads=hq, dim=dim, page=16, extra_pages=1, spare=8, seed=4)
    used = set(p.table[p.table >= 0].cpu().tolist())
    free = [i for i in range(p.n_pages) if i not in used]
    freq = vm.RopeFrequencies(dim)
    handle, scratch = vm.Rope.Create(rt, dim, hq, hk, "bf16", frequencies=freq), vm.Scratch.Create(rt)
    stream = torch.cuda.Stream()

    def product(lp, a, b, n, m):
        out = torch.empty((n, m), dtype=torch.bfloat16, device="cuda")
        lp.ExecuteDeviceAsync([a.data_ptr(), b.data_ptr()], [out.data_ptr()], stream.cuda_stream)
        return out

    def check_product(a, b, got):
        want, size = a.double() @ b.double(), a.double().abs() @ b.double().abs()
        assert bool(((got.double() - want).abs() <= half_step("bf16") * want.abs() + a.shape[1] * U * size).all())

    def forward(x, rows):
        n = sum(rows)
        lp_in, lp_out = programs[n]
        pos = torch.cat([torch.arange(length - k, length, dtype=torch.int32) for k, length in zip(rows, p.lengths)]).cuda()
        attended = torch.empty((n, hq, dim), dtype=torch.bfloat16, device="cuda")
        turned = [torch.empty((n, h, dim), dtype=torch.bfloat16, device="cuda") for h in (hq, hk)]
        torch.cuda.synchronize()
        qkv = product(lp_in, x, w_in, n, wide)
        q, k, v = qkv.view(n, -1, dim).split((hq, hk, hk), 1)
        handle.Apply(n, pos.data_ptr(), vm.Rows.Of(q), vm.Rows.Of(k), *map(vm.Rows.Of, turned), stream=stream.cuda_stream)
        p.cache.Write(p.batch, vm.Rows.Of(turned[1]), vm.Rows.Of(v), stream=stream.cuda_stream)
        p.cache.Attend(p.batch, vm.Rows.Of(turned[0]), vm.Rows.Of(attended), scratch, stream=stream.cuda_stream)
        y = product(lp_out, attended, w_out, n, width)
        torch.cuda.synchronize()
        assert p.cache.Status()["code"] == 0 and lp_in.Status()["code"] == 0 and lp_out.Status()["code"] == 0
        check_product(x, w_in, qkv)
        for t, got in ((q, turned[0]), (k, turned[1])):
            want = rope(t.double(), None, pos, freq, dim, False, False, 0.0, 1.0)
            assert bool(((got.double() - want).abs() <= half_step("bf16") * want.abs() + 12 * U * t.double().abs().amax(-1, keepdim=True)).all())
        if cache == "bf16":                               # (the new rows are in the pages as they are; those of 8 bits to half a step of 2^-3)
            places = p.places()
            i, page, slot = (torch.tensor(c, device="cuda") for c in zip(*places))
            assert torch.equal(p.pages[0][page, slot], turned[1][i]) and torch.equal(p.pages[1][page, slot], v[i])
        want, _, tol = p.attend(turned[0], dim ** -0.5)
        assert bool(((attended.double() - want).abs() <= tol + half_step("bf16") * want.abs()).all())
        check_product(attended.view(n, -1), w_out, y)

    forward(x0[:total].contiguous(), prompts)
    p.rows, p.max_rows, p.total, p.n_rows = [1] * len(prompts), 1, len(prompts), len(prompts)
    p.start = torch.arange(len(prompts) + 1, dtype=torch.int32, device="cuda")
    p.bind()
    for s in range(steps):
        for b in range(len(prompts)):
            p.lengths[b] += 1
            e = (p.lengths[b] - 1) // p.page
            if int(p.table[b, e]) < 0:
                p.table[b, e] = free.pop()
        p.length.copy_(torch.tensor(p.lengths, dtype=torch.int32))
        forward(x0[total + s * len(prompts):total + (s + 1) * len(prompts)].contiguous(), p.rows)
