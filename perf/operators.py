"""The attention operators beside the programs, as calls to be timed: rotary positions with the norms of queries and keys
(forward and backward), the paged cache (written, read back) and the attention of new rows over it.

`own` False: the operators in elementary torch operations, in 32 bits (angles in 64), rounded once. `own` True: the calls of
this package. Both take the same inputs.
"""
import importlib
import math
import random

import torch

own = False

_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1}
_EPS = 1e-6


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def listed():
    return [
        # the rotation of one decode step: 32 sequences, 16 heads of 64, as the decode program here has them
        {"name": "rotate_step", "op": "rotate", "rows": 32, "q_heads": 16, "k_heads": 16, "dim": 64, "rot": 64, "dtype": "bf16",
         "norm": False, "interleaved": False, "scaling": "plain", "factor": 1.0, "far": 2049},
        # a whole prompt batch (8 x 2048 rows) of a model with norms of queries and keys and a stretched context
        {"name": "rotate_prompt", "op": "rotate", "rows": 16384, "q_heads": 32, "k_heads": 8, "dim": 128, "rot": 128, "dtype": "bf16",
         "norm": True, "interleaved": False, "scaling": "parts", "factor": 4.0, "far": 131072},
        # the same in a training step's backward pass, one row short of a round number
        {"name": "rotate_back", "op": "rotate_back", "rows": 8191, "q_heads": 32, "k_heads": 8, "dim": 128, "rot": 128, "dtype": "bf16",
         "norm": True, "interleaved": False, "scaling": "plain", "factor": 1.0, "far": 8192},
        # f32 training of a small model: neighbouring pairs, half of a head of 96, an odd number of rows
        {"name": "rotate_back_odd", "op": "rotate_back", "rows": 1777, "q_heads": 12, "k_heads": 4, "dim": 96, "rot": 48, "dtype": "f32",
         "norm": True, "interleaved": True, "scaling": "linear", "factor": 2.0, "far": 4096},
        # one decode step's keys and values into an 8-bit cache
        {"name": "write_step", "op": "write", "seqs": 32, "rows_lo": 1, "rows_hi": 1, "past_lo": 100, "past_hi": 2048, "pad": 0,
         "k_heads": 8, "dim": 128, "dtype": "bf16", "cache": "e4m3", "page": 64, "mix": 1},
        # eight prompts of different lengths into an 8-bit cache, in a batch padded to its bucket
        {"name": "write_prompt", "op": "write", "seqs": 8, "rows_lo": 500, "rows_hi": 3500, "past_lo": 0, "past_hi": 500, "pad": 300,
         "k_heads": 8, "dim": 128, "dtype": "bf16", "cache": "e4m3", "page": 64, "mix": 2},
        # sixteen cached sequences taken back whole, as when they move to another cache
        {"name": "read_whole", "op": "read", "seqs": 16, "rows_lo": 300, "rows_hi": 8000, "past_lo": 0, "past_hi": 0, "pad": 0,
         "k_heads": 8, "dim": 128, "dtype": "bf16", "cache": "e4m3", "page": 64, "mix": 3},
        # the last rows of a few sequences, 16-bit pages of an odd size, heads of 80
        {"name": "read_odd", "op": "read", "seqs": 5, "rows_lo": 30, "rows_hi": 1200, "past_lo": 0, "past_hi": 300, "pad": 0,
         "k_heads": 4, "dim": 80, "dtype": "f16", "cache": "f16", "page": 24, "mix": 4},
        # one token of one short sequence: latency
        {"name": "attend_first", "op": "attend", "seqs": 1, "rows_lo": 1, "rows_hi": 1, "past_lo": 300, "past_hi": 300, "pad": 0,
         "q_heads": 32, "k_heads": 8, "dim": 128, "dtype": "bf16", "cache": "bf16", "page": 64, "window": 0, "mix": 5},
        # one decode step of 64 sequences of 200 to 16000 tokens over an 8-bit cache
        {"name": "attend_steps", "op": "attend", "seqs": 64, "rows_lo": 1, "rows_hi": 1, "past_lo": 200, "past_hi": 16000, "pad": 0,
         "q_heads": 32, "k_heads": 8, "dim": 128, "dtype": "bf16", "cache": "e4m3", "page": 64, "window": 0, "mix": 6},
        # a prompt's chunk of 2048 behind 14336 cached tokens
        {"name": "attend_chunk", "op": "attend", "seqs": 1, "rows_lo": 2048, "rows_hi": 2048, "past_lo": 14336, "past_hi": 14336, "pad": 0,
         "q_heads": 32, "k_heads": 8, "dim": 128, "dtype": "bf16", "cache": "bf16", "page": 64, "window": 0, "mix": 7},
        # chunks and single tokens in one padded batch, 16 heads of 64, a sliding window, pages that no tile divides
        {"name": "attend_mixed", "op": "attend", "seqs": 12, "rows_lo": 1, "rows_hi": 1500, "past_lo": 0, "past_hi": 4000, "pad": 77,
         "q_heads": 16, "k_heads": 16, "dim": 64, "dtype": "f16", "cache": "f16", "page": 48, "window": 1000, "mix": 8},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(max(lo, 1)), math.log(max(hi, 1)) + 1e-9))))) if hi > 0 else 0


def draw(rng):
    op = rng.choice(["rotate", "rotate_back", "write", "read", "attend", "attend", "attend"])
    if op in ("rotate", "rotate_back"):
        dim = rng.choice([32, 64, 80, 96, 128, 128, 256])
        k_heads = rng.choice([1, 2, 4, 8, 16])
        c = {"op": op, "q_heads": k_heads * rng.choice([1, 2, 4, 5]), "k_heads": k_heads, "dim": dim, "rot": rng.choice([dim, dim, dim // 2]),
             "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]), "norm": rng.random() < 0.7, "interleaved": rng.random() < 0.4,
             "scaling": rng.choice(["plain", "linear", "stretch", "parts"]), "far": _log(rng, 64, 1000000)}
        c["factor"] = 1.0 if c["scaling"] == "plain" else rng.choice([2.0, 8.0])
        c["rows"] = _log(rng, 1, min(16384, 20000000 * 2 // ((c["q_heads"] + k_heads) * dim * _SIZE[c["dtype"]])))
        return c
    while True:
        dim, k_heads = rng.choice([64, 80, 128, 128]), rng.choice([1, 2, 4, 8, 16])
        c = {"op": op, "seqs": _log(rng, 1, 64), "rows_lo": 1, "rows_hi": 1, "past_lo": _log(rng, 1, 300), "past_hi": _log(rng, 300, 16000),
             "pad": rng.choice([0, 0, 5, 131]), "k_heads": k_heads, "dim": dim, "dtype": rng.choice(["bf16", "f16"]),
             "page": rng.choice([16, 24, 32, 64, 128, 256]), "mix": rng.randrange(1 << 30)}
        c["cache"] = rng.choice([c["dtype"], "e4m3"])
        if op != "attend" or rng.random() < 0.6:
            c["rows_hi"] = _log(rng, 1, 4000)
            c["rows_lo"] = max(1, c["rows_hi"] // rng.choice([1, 4, 50]))
        if op == "attend":
            c["q_heads"] = k_heads * rng.choice([1, 2, 4, 7, 8])
            c["window"] = rng.choice([0, 0, 0, _log(rng, 16, 4000)])
        rows, lengths = _lengths(c)
        w = work(c)
        if w["bytes"] > 4e8 or w["flops"] > 2.5e11 or sum(lengths) * k_heads * dim > 1.2e8:
            continue
        if op == "attend" and len(rows) * max(rows) * max(lengths) * c["q_heads"] > 1.2e9 or len(rows) * max(lengths) * k_heads * dim * (c.get("q_heads", 0) + 8) > 3e10:
            continue
        return c


def _lengths(case):
    """New rows and whole length of each sequence."""
    rng = random.Random(case["mix"])
    rows = [_log(rng, case["rows_lo"], case["rows_hi"]) for _ in range(case["seqs"])]
    return rows, [n + _log(rng, case["past_lo"], case["past_hi"]) for n in rows]


def _seen(n, length, window):
    """Keys that the rows of a sequence see: of all of them together, and counted for each row."""
    pairs = 0
    for i in range(n):
        p = length - n + i
        pairs += min(p + 1, window) if window else p + 1
    first = max(0, length - n - window + 1) if window else 0
    return length - first, pairs


def work(case):
    if case["op"] in ("rotate", "rotate_back"):
        elems = case["rows"] * (case["q_heads"] + case["k_heads"]) * case["dim"]
        passes = 2 if case["op"] == "rotate" or not case["norm"] else 3
        weights = 2 * 4 * case["dim"] * (2 if case["op"] == "rotate_back" else 1) if case["norm"] else 0
        return {"bytes": passes * elems * _SIZE[case["dtype"]] + 4 * case["rows"] + weights, "flops": elems * (10 if passes == 3 else 5)}
    rows, lengths = _lengths(case)
    row = case["k_heads"] * case["dim"]
    if case["op"] in ("write", "read"):
        scales = 8 * case["k_heads"] if case["cache"] == "e4m3" else 0
        return {"bytes": sum(rows) * (2 * row * (_SIZE[case["dtype"]] + _SIZE[case["cache"]]) + scales), "flops": sum(rows) * row * 4}
    seen = [_seen(n, length, case["window"]) for n, length in zip(rows, lengths)]
    per_key = 2 * row * _SIZE[case["cache"]] + (8 * case["k_heads"] if case["cache"] == "e4m3" else 0)
    q = sum(rows) * case["q_heads"] * (2 * case["dim"] * _SIZE[case["dtype"]] + 4)
    return {"bytes": q + per_key * sum(k for k, _ in seen), "flops": 4 * case["dim"] * case["q_heads"] * sum(p for _, p in seen)}


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _frequencies(rot, scaling, factor, original=4096.0, base=10000.0):
    i = torch.arange(0, rot, 2, dtype=torch.float64, device="cuda")
    if scaling == "stretch" and rot > 2:
        base = base * factor ** (rot / (rot - 2))
    f = base ** (-i / max(rot, 1))
    if scaling == "linear":
        f = f / factor
    elif scaling == "parts":       # as many turns as `fast` over the original length stay, as few as `slow` are slowed down
        keep = ((original * f / (2 * math.pi) - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        f = f * (keep + (1 - keep) / factor)
    return f


def _magnitude(case):
    return 0.1 * math.log(case["factor"]) + 1.0 if case["scaling"] == "parts" else 1.0


def _normal(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def _quantise(x):
    s = x.abs().amax(-1) / torch.full((), 448.0, device=x.device)
    codes = torch.where(s[..., None] > 0, x / s[..., None], torch.zeros((), device=x.device)).clamp(-448.0, 448.0)
    return codes.to(torch.float8_e4m3fn), s


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DT[case["dtype"]]
    s = {"op": case["op"], "case": case}
    if case["op"] in ("rotate", "rotate_back"):
        n, hq, hk, d = case["rows"], case["q_heads"], case["k_heads"], case["dim"]
        qkv = _normal(gen, (n, (hq + 2 * hk) * d), dt, 1.5)           # a fused projection's result; queries and keys are views of it
        s["q"], s["k"] = qkv[:, :hq * d].view(n, hq, d), qkv[:, hq * d:(hq + hk) * d].view(n, hk, d)
        s["position"] = torch.randint(0, case["far"], (n,), generator=gen, device="cuda", dtype=torch.int32)
        s["frequency"] = _frequencies(case["rot"], case["scaling"], case["factor"])
        if case["norm"]:
            s["qw"], s["kw"] = (1.0 + 0.2 * torch.randn(d, generator=gen, device="cuda") for _ in range(2))
        if case["op"] == "rotate_back":
            s["dq"], s["dk"] = _normal(gen, (n, hq, d), dt), _normal(gen, (n, hk, d), dt)
        s["out"] = [torch.empty(n, h, d, dtype=dt, device="cuda") for h in (hq, hk)]
        if case["op"] == "rotate_back" and case["norm"]:
            s["out"] += [torch.empty(d, device="cuda") for _ in range(2)]
        if own:
            _bind_rope(s)
        return s
    rows, lengths = _lengths(case)
    hk, d, ps, cache = case["k_heads"], case["dim"], case["page"], _DT[case["cache"]]
    pages = [-(-length // ps) for length in lengths]
    n_pages = sum(pages) + 3
    order = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros(len(rows), max(pages), dtype=torch.int32)
    at = 0
    host_order = order.cpu()
    for b, p in enumerate(pages):
        table[b, :p] = host_order[at:at + p]
        at += p
    s["table"] = table.cuda()
    start = [0]
    for n in rows:
        start.append(start[-1] + n)
    s["start"] = torch.tensor(start, dtype=torch.int32, device="cuda")
    s["length"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    s["total"], s["n_rows"], s["max_rows"], s["max_length"] = start[-1], start[-1] + case["pad"], max(rows), max(lengths)
    for name in ("k", "v"):
        x = _normal(gen, (n_pages, ps, hk, d), dt)
        if case["cache"] == "e4m3":
            s[name + "_pages"], s[name + "_scales"] = _quantise(x.float())
        else:
            s[name + "_pages"] = x
    if case["op"] == "write":
        s["k"], s["v"] = (_normal(gen, (s["n_rows"], hk, d), dt) for _ in range(2))
    elif case["op"] == "read":
        s["out"] = [torch.empty(s["n_rows"], hk, d, dtype=dt, device="cuda") for _ in range(2)]
    else:
        s["q"] = _normal(gen, (s["n_rows"], case["q_heads"], d), dt, 2.0)
        s["out"] = [torch.empty_like(s["q"]), torch.empty(s["n_rows"], case["q_heads"], device="cuda")]
    if own:
        _bind_cache(s)
    return s


# ---------------------------------------------------------------------------------------------
# the package's calls
# ---------------------------------------------------------------------------------------------
_rt = _scratch = None


def _package():
    global _rt, _scratch
    vm = importlib.import_module("pjrt-ocl_b200")
    if _rt is None:
        _rt = vm.Runtime.Create(torch.cuda.current_device())
        _scratch = vm.Scratch.Create(_rt)
    return vm, _rt


def _bind_rope(s):
    vm, rt = _package()
    c = s["case"]
    s["rope"] = vm.Rope.Create(rt, head_dim=c["dim"], rot_dim=c["rot"], q_heads=c["q_heads"], k_heads=c["k_heads"], dtype=c["dtype"],
                               interleaved=c["interleaved"], norm=c["norm"], eps=_EPS, magnitude=_magnitude(c),
                               frequencies=vm.RopeFrequencies(c["rot"], 10000.0, c["scaling"], c["factor"], 4096.0, 1.0, 32.0))
    s["rows"] = [vm.Rows.Of(t) for t in (s["q"], s["k"], *([s["dq"], s["dk"]] if c["op"] == "rotate_back" else []), *s["out"][:2])]
    s["p"] = [s["position"].data_ptr()] + [t.data_ptr() for t in ([s["qw"], s["kw"]] if c["norm"] else [])] + [t.data_ptr() for t in s["out"][2:]]
    s["p"] += [0] * (5 - len(s["p"]))


def _bind_cache(s):
    vm, rt = _package()
    c = s["case"]
    scales = [s[n].data_ptr() for n in ("k_scales", "v_scales") if n in s] or [0, 0]
    s["cache"] = vm.PagedCache.Create(rt, dtype=c["cache"], row_dtype=c["dtype"], heads=c["k_heads"], q_heads=c.get("q_heads", c["k_heads"]), head_dim=c["dim"],
                                      page_size=c["page"], n_pages=s["k_pages"].shape[0], k_pages=s["k_pages"].data_ptr(), v_pages=s["v_pages"].data_ptr(),
                                      k_scales=scales[0], v_scales=scales[1])
    s["batch"] = vm.Batch(n_seqs=c["seqs"], row_start=s["start"].data_ptr(), length=s["length"].data_ptr(), pages=s["table"].data_ptr(),
                          max_pages=s["table"].shape[1], n_rows=s["n_rows"], max_rows=s["max_rows"])
    s["rows"] = [vm.Rows.Of(t) for t in ([s["k"], s["v"]] if c["op"] == "write" else s["out"] if c["op"] == "read" else [s["q"], s["out"][0]])]


def _own(s):
    stream = torch.cuda.current_stream().cuda_stream
    op, c, r = s["op"], s["case"], s["rows"]
    if op == "rotate":
        s["rope"].Apply(c["rows"], s["p"][0], r[0], r[1], r[2], r[3], q_weight=s["p"][1], k_weight=s["p"][2], stream=stream)
        return s["out"]
    if op == "rotate_back":
        s["rope"].ApplyBackward(c["rows"], s["p"][0], r[0], r[1], r[2], r[3], r[4], r[5], q_weight=s["p"][1], k_weight=s["p"][2],
                                dq_weight=s["p"][3], dk_weight=s["p"][4], scratch=_scratch, stream=stream)
        return s["out"]
    if op == "write":
        s["cache"].Write(s["batch"], r[0], r[1], stream=stream)
        return [s[n] for n in ("k_pages", "v_pages", "k_scales", "v_scales") if n in s]
    if op == "read":
        s["cache"].Read(s["batch"], r[0], r[1], stream=stream)
        return [t[:s["total"]] for t in s["out"]]
    s["cache"].Attend(s["batch"], r[0], r[1], _scratch, lse=s["out"][1].data_ptr(), scale=c["dim"] ** -0.5, causal=True, window=c["window"], stream=stream)
    return [t[:s["total"]] for t in s["out"]]


# ---------------------------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------------------------
def _cos_sin(s):
    angle = s["position"].double()[:, None] * s["frequency"]
    m = _magnitude(s["case"])
    return (torch.cos(angle) * m).float()[:, None], (torch.sin(angle) * m).float()[:, None]


def _halves(y, c):
    rot = c["rot"]
    if c["interleaved"]:
        return y[..., 0:rot:2], y[..., 1:rot:2], y[..., rot:]
    return y[..., :rot // 2], y[..., rot // 2:rot], y[..., rot:]


def _joined(a, b, rest, c):
    front = torch.stack((a, b), -1).flatten(-2) if c["interleaved"] else torch.cat((a, b), -1)
    return torch.cat((front, rest), -1)


def _rotate(x, w, cos, sin, c):
    y = x.float()
    if c["norm"]:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + _EPS) * w
    a, b, rest = _halves(y, c)
    return _joined(a * cos - b * sin, a * sin + b * cos, rest, c).to(x.dtype)


def _rotate_back(x, w, dy, cos, sin, c):
    a, b, rest = _halves(dy.float(), c)
    g = _joined(a * cos + b * sin, b * cos - a * sin, rest, c)
    if not c["norm"]:
        return g.to(dy.dtype), None
    x = x.float()
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS)
    h = g * w
    dx = r * h - x * (r * r * r * (h * x).mean(-1, keepdim=True))
    return dx.to(dy.dtype), (g * x * r).sum((0, 1))


def _places(s):
    """Page and slot of each new row."""
    i = torch.arange(s["total"], device="cuda", dtype=torch.int32)
    b = torch.searchsorted(s["start"], i, right=True) - 1
    pos = (s["length"][b] - s["start"][b + 1] + i).long()
    ps = s["case"]["page"]
    return s["table"][b, pos // ps].long(), pos % ps


def _write(s):
    page, slot = _places(s)
    for name in ("k", "v"):
        x = s[name][:s["total"]]
        if s["case"]["cache"] == "e4m3":
            codes, scales = _quantise(x.float())
            s[name + "_pages"].view(torch.uint8)[page, slot] = codes.view(torch.uint8)
            s[name + "_scales"][page, slot] = scales
        else:
            s[name + "_pages"][page, slot] = x
    return [s[n] for n in ("k_pages", "v_pages", "k_scales", "v_scales") if n in s]


def _values(s, name, page, slot):
    """Rows of the cache as f32."""
    if s["case"]["cache"] != "e4m3":
        return s[name + "_pages"][page, slot].float()
    return s[name + "_pages"].view(torch.uint8)[page, slot].view(torch.float8_e4m3fn).float() * s[name + "_scales"][page, slot][..., None]


def _read(s):
    page, slot = _places(s)
    return [_values(s, name, page, slot).to(_DT[s["case"]["dtype"]]) for name in ("k", "v")]


def _attend(s):
    """All sequences at once, padded to the longest."""
    c = s["case"]
    hk, d, n, ln = c["k_heads"], c["dim"], s["max_rows"], s["max_length"]
    pos = torch.arange(ln, device="cuda")
    page, slot = s["table"].long()[:, pos // c["page"]], (pos % c["page"]).expand(c["seqs"], ln)
    k, v = _values(s, "k", page, slot), _values(s, "v", page, slot)                      # [seqs, ln, hk, d]
    rows = (s["start"][1:] - s["start"][:-1]).long()
    i = torch.arange(n, device="cuda")
    live = i < rows[:, None]
    at = torch.where(live, s["start"][:-1, None] + i, torch.zeros((), dtype=torch.int64, device="cuda"))
    q = s["q"][at].float().view(c["seqs"], n, hk, -1, d).permute(0, 2, 3, 1, 4)          # [seqs, hk, group, n, d]
    p = torch.matmul(q.reshape(c["seqs"], hk, -1, d), k.permute(0, 2, 3, 1)).view(c["seqs"], hk, -1, n, ln)
    where = (s["length"].long()[:, None] - rows[:, None] + i)[:, :, None]                # position of each row
    hidden = pos > where
    if c["window"]:
        hidden = hidden | (pos <= where - c["window"])
    p = p.mul_(d ** -0.5).masked_fill_(hidden[:, None, None], float("-inf"))
    top = p.amax(-1, keepdim=True)
    p = p.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(c["seqs"], hk, -1, ln), v.permute(0, 2, 1, 3)).view(c["seqs"], hk, -1, n, d) / total
    lse = (top + total.log())[..., 0].permute(0, 3, 1, 2).flatten(2)                     # [seqs, n, heads]
    return [out.permute(0, 3, 1, 2, 4).flatten(2, 3)[live].to(s["q"].dtype), lse[live]]


def _plain(s):
    c = s["case"]
    if s["op"] in ("rotate", "rotate_back"):
        cos, sin = _cos_sin(s)
        if s["op"] == "rotate":
            return [_rotate(s["q"], s.get("qw"), cos, sin, c), _rotate(s["k"], s.get("kw"), cos, sin, c)]
        (dq, wq), (dk, wk) = (_rotate_back(s[x], s.get(x + "w"), s["d" + x], cos, sin, c) for x in ("q", "k"))
        return [dq, dk] + ([wq, wk] if c["norm"] else [])
    return {"write": _write, "read": _read, "attend": _attend}[s["op"]](s)


def run(s):
    return _own(s) if own else _plain(s)


# ---------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------
def _turned(x, w, turn, c):
    """Norm and rotation of x [rows, heads, dim] as products of complex numbers."""
    if c["norm"]:
        x = x / ((x ** 2).sum(-1, keepdim=True) / c["dim"] + _EPS).sqrt() * w
    half = c["rot"] // 2
    if c["interleaved"]:
        z = torch.view_as_complex(x[..., :c["rot"]].unflatten(-1, (half, 2)).contiguous()) * turn
        return torch.cat((torch.view_as_real(z).flatten(-2), x[..., c["rot"]:]), -1)
    z = torch.complex(x[..., :half], x[..., half:c["rot"]]) * turn
    return torch.cat((z.real, z.imag, x[..., c["rot"]:]), -1)


def _cached(s, b, length):
    """K and V of sequence b, in 64 bits, heads first."""
    ps = s["case"]["page"]
    page = s["table"][b, :-(-length // ps)].long()
    got = []
    for name in ("k", "v"):
        x = s[name + "_pages"].view(torch.uint8)[page].view(s[name + "_pages"].dtype).double()
        if name + "_scales" in s:
            x = x * s[name + "_scales"][page].double()[..., None]
        got.append(x.flatten(0, 1)[:length].transpose(0, 1))
    return got


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("rotate", "rotate_back"):
        angle = torch.outer(s["position"].double(), s["frequency"])
        turn = torch.polar(torch.full_like(angle, _magnitude(case)), angle)[:, None]
        got = []
        for x in ("q", "k"):
            v = s[x].double()
            w = s[x + "w"].double() if case["norm"] else None
            if case["op"] == "rotate":
                got.append([_turned(v, w, turn, case)])
                continue
            leaves = [t.requires_grad_() for t in ([v, w] if case["norm"] else [v])]
            with torch.enable_grad():
                got.append(torch.autograd.grad(_turned(v, w, turn, case), leaves, s["d" + x].double()))
        return [g[0] for g in got] + [g[1] for g in got if len(g) > 1]
    rows, lengths = _lengths(case)
    if case["op"] == "write":
        if case["cache"] != "e4m3":
            return None
        want = []
        for name in ("k", "v"):
            scales = s[name + "_scales"].double()
            flat, i = s[name].double().abs().amax(-1) / 448.0, 0
            for b, (n, length) in enumerate(zip(rows, lengths)):
                at = torch.arange(length - n, length, device="cuda")
                scales[s["table"][b, at // case["page"]].long(), at % case["page"]] = flat[i:i + n]
                i += n
            want.append(scales)
        return [None, None, *want]
    out = [[], []]
    for b, (n, length) in enumerate(zip(rows, lengths)):
        k, v = _cached(s, b, length)
        if case["op"] == "read":
            out[0].append(k[:, length - n:].transpose(0, 1))
            out[1].append(v[:, length - n:].transpose(0, 1))
            continue
        first = int(s["start"][b])
        q = s["q"][first:first + n].double().transpose(0, 1)
        group = q.shape[0] // k.shape[0]
        position = torch.arange(length - n, length, device="cuda")[:, None]
        key = torch.arange(length, device="cuda")[None]
        seen = (key <= position) & (key > position - case["window"]) if case["window"] else key <= position
        o, e = [], []
        for h in range(q.shape[0]):
            score = (q[h] @ k[h // group].T / math.sqrt(case["dim"])).masked_fill(~seen, float("-inf"))
            e.append(torch.logsumexp(score, -1))
            o.append(torch.softmax(score, -1) @ v[h // group])
        out[0].append(torch.stack(o, 1))
        out[1].append(torch.stack(e, 1))
    return [torch.cat(x) for x in out]
