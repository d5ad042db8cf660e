"""Plain forms of the operators in 64 bits, and inputs for them (pages in a shuffled order, ragged batches)."""
from __future__ import annotations

import torch

from conftest import package

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
U = 2.0 ** -24                         # half a step of f32


def half_step(dtype):
    return torch.finfo(DT[dtype]).eps / 2


def normal(shape, dtype, seed, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(DT[dtype] if isinstance(dtype, str) else dtype)


# ---- rotary positions ----
def rope(x, w, positions, freq, rot, interleaved, norm, eps, magnitude):
    """x [rows, heads, dim] in 64 bits."""
    if norm:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps)
        if w is not None:
            x = x * w
    angle = positions.double()[:, None] * torch.tensor(freq, dtype=torch.float64, device=x.device)
    cos, sin = (torch.cos(angle) * magnitude)[:, None], (torch.sin(angle) * magnitude)[:, None]
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((y, x[..., rot:]), -1)


# ---- the cache ----
def quantised(x):
    """Codes and scales of f32 rows, by the definition (both divisions in f32)."""
    s = x.abs().amax(-1) / torch.full((), 448.0, device=x.device)
    y = torch.where(s[..., None] == 0, torch.zeros((), device=x.device), x / s[..., None])
    return y.clamp(-448.0, 448.0).to(torch.float8_e4m3fn), s


class Paged:
    """A cache with its batch: sequences of `rows` new rows behind `past` positions, on pages in a shuffled order."""

    def __init__(self, rt, rows, past, *, dtype="bf16", row_dtype=None, heads=2, q_heads=None, dim=64, page=16, seed=0, spare=2, head_major=False, pad=0,
                 max_rows=None, lengths=None, extra_pages=0):
        vm = package()
        self.vm, self.rt = vm, rt
        self.rows, self.lengths = list(rows), [n + p for n, p in zip(rows, past)] if lengths is None else list(lengths)
        self.dtype, self.row_dtype = dtype, row_dtype or ("bf16" if dtype == "e4m3" else dtype)
        self.heads, self.q_heads, self.dim, self.page = heads, q_heads or heads, dim, page
        need = [-(-n // page) for n in self.lengths]
        self.n_pages = sum(need) + spare
        gen = torch.Generator(device="cuda").manual_seed(seed + 77)
        order = torch.randperm(self.n_pages, generator=gen, device="cuda").to(torch.int32).cpu()
        cols = max([1, *need]) + extra_pages
        table = torch.full((max(1, len(rows)), cols), -7, dtype=torch.int32)       # entries behind a sequence's own are not read
        at = 0
        for b, k in enumerate(need):
            table[b, :k] = order[at:at + k]
            at += k
        self.table = table.cuda()
        start = [0]
        for n in rows:
            start.append(start[-1] + n)
        self.total, self.n_rows = start[-1], start[-1] + pad
        self.start = torch.tensor(start, dtype=torch.int32, device="cuda")
        self.length = torch.tensor(self.lengths or [0], dtype=torch.int32, device="cuda")
        shape = (self.n_pages, heads, page, dim) if head_major else (self.n_pages, page, heads, dim)
        self.pages, self.scales = [], [None, None]
        for i in range(2):
            x = normal(shape, "f32", seed + i)
            if head_major:
                x = x.transpose(1, 2)
            if dtype == "e4m3":
                codes, s = quantised(x)
                codes = codes.view(torch.uint8)
                if head_major:
                    codes = codes.transpose(1, 2).contiguous().transpose(1, 2)
                self.pages.append(codes.view(torch.float8_e4m3fn))
                self.scales[i] = s.contiguous()
            else:
                self.pages.append(x.to(DT[dtype]))
        self.max_rows = max([0, *rows]) if max_rows is None else max_rows
        self.bind()

    def bind(self):
        vm = self.vm
        k, v = self.pages
        ss = {} if self.scales[0] is None else {"k_scales": self.scales[0].data_ptr(), "v_scales": self.scales[1].data_ptr(), "scale_strides": self.scales[0].stride()}
        self.cache = vm.PagedCache.Create(self.rt, dtype=self.dtype, row_dtype=self.row_dtype, heads=self.heads, q_heads=self.q_heads, head_dim=self.dim, page_size=self.page,
                                          n_pages=self.n_pages, k_pages=k.data_ptr(), v_pages=v.data_ptr(), strides=k.stride()[:3], **ss)
        self.batch = vm.Batch(len(self.rows), self.start.data_ptr(), self.length.data_ptr(), self.table.data_ptr(), self.table.shape[1], self.n_rows, self.max_rows)

    def places(self):
        """(row, page, slot) of every new row that has a position."""
        out = []
        i = 0
        for b, (n, length) in enumerate(zip(self.rows, self.lengths)):
            for p in range(length - n, length):
                if p >= 0:
                    out.append((i, int(self.table[b, p // self.page]), p % self.page))
                i += 1
        return out

    def values(self, b, which, lo=0):
        """Positions of sequence b in 64 bits: [position, head, dim]."""
        pos = torch.arange(lo, self.lengths[b], device="cuda")
        page, slot = self.table[b, pos // self.page].long(), pos % self.page
        x = self.pages[which]
        if self.dtype == "e4m3":
            return x.view(torch.uint8)[page, slot].view(torch.float8_e4m3fn).double() * self.scales[which][page, slot].double()[..., None]
        return x[page, slot].double()

    def attend(self, q, scale, causal=True, window=0):
        """out, lse, and how far f32 sums and 16-bit weights may be off, for the batch's rows; nothing for those behind the last."""
        outs, lses, tols = [], [], []
        i = 0
        g = self.q_heads // self.heads
        p_step = half_step("f16" if self.dtype == "e4m3" else self.row_dtype)
        for b, (n, length) in enumerate(zip(self.rows, self.lengths)):
            k, v = (self.values(b, w).repeat_interleave(g, 1).transpose(0, 1) for w in (0, 1))       # [heads, length, dim]
            x = q[i:i + n].double().transpose(0, 1)
            i += n
            row, key = torch.arange(length - n, length, device="cuda")[:, None], torch.arange(length, device="cuda")[None]
            seen = (key <= row) if causal else torch.ones_like(key <= row)
            if window:
                seen = seen & (key > row - window)
            s = (x @ k.transpose(1, 2) * scale).masked_fill(~seen, float("-inf"))
            top = s.amax(-1, keepdim=True) if length else torch.full((*s.shape[:2], 1), float("-inf"), dtype=torch.float64, device="cuda")
            e = torch.where(seen, torch.exp(s - torch.where(torch.isfinite(top), top, torch.zeros_like(top))), torch.zeros_like(s))
            total = e.sum(-1, keepdim=True)
            w = torch.where(total > 0, e / total, torch.zeros_like(e))
            v0 = torch.where(torch.isfinite(v), v, torch.zeros_like(v))
            outs.append((w @ v0).transpose(0, 1))
            lses.append((torch.where(torch.isfinite(top), top, torch.zeros_like(top)) + total.log())[..., 0].T)
            # a score is off by dim roundings of sum |q k|; a weight by that, by the exponential (2^-22) and by its 16 bits, the
            # sums by a rounding for each key; all of it relative to sum w |v|
            reach = ((x.abs() @ k.abs().transpose(1, 2)) * scale).masked_fill(~seen, 0.0).amax(-1, keepdim=True) if length else torch.zeros_like(total)
            off = 2 * ((self.dim + 4) * U * reach + 2.0 ** -22 + (length / 8 + 16) * U) + p_step
            tols.append((off * (w @ v0.abs())).transpose(0, 1))
        cat = lambda x, shape: torch.cat(x) if x else torch.zeros(shape, dtype=torch.float64, device="cuda")  # noqa: E731
        return cat(outs, (0, self.q_heads, self.dim)), cat(lses, (0, self.q_heads)), cat(tols, (0, self.q_heads, self.dim))
