"""Tensors given to the operators beside the programs in place of addresses: what is checked, without a device; and the same results."""
import pytest

torch = pytest.importorskip("torch")

from conftest import package  # noqa: E402


class OnDevice:
    """What the checks look at, of a tensor on a device."""

    def __init__(self, *shape, dtype=torch.int32, index=0, strided=False):
        self._t = torch.zeros(*shape, dtype=dtype)
        if strided:
            self._t = torch.zeros(*shape[:-1], 2 * shape[-1], dtype=dtype)[..., ::2]
        self.dtype, self.shape, self.is_cuda, self.device = dtype, self._t.shape, True, torch.device("cuda", index)
        self.dim, self.numel, self.stride, self.is_contiguous = self._t.dim, self._t.numel, self._t.stride, self._t.is_contiguous

    def data_ptr(self):
        return 4096


def test_batches_of_tensors():
    vm = package()
    t = OnDevice
    good = dict(n_seqs=2, row_start=t(3), length=t(2), pages=t(2, 5), max_pages=4, n_rows=7)
    b = vm.Batch(**good)
    assert (b._keep.row_start, b._keep.length, b._keep.pages, b._keep.pages_stride, b._keep.max_pages) == (4096, 4096, 4096, 5, 4)
    assert vm.Batch(2, 4096, 4096, 8192, 4, 7)._keep.pages_stride == 4               # (addresses are taken as they are)
    assert vm.Batch(0, None, None, None, 0, 3)._keep.pages is None
    for change, part in ((dict(row_start=t(3, dtype=torch.int64)), "row_start: of type torch.int64"), (dict(length=t(2, dtype=torch.float32)), "length: of type"),
                         (dict(pages=t(2, 5, dtype=torch.int64)), "pages: of type"), (dict(row_start=t(2)), "row_start: .* want 3 values"), (dict(length=t(1)), "length: .* want 2"),
                         (dict(pages=t(1, 5)), "pages: .* want 9"), (dict(pages=t(2, 5, strided=True)), "without gaps"), (dict(length=t(2, index=1)), "length: on cuda:1"),
                         (dict(length=torch.zeros(2, dtype=torch.int32)), "length: on cpu"), (dict(max_pages=6), "pages: .* want 11")):
        with pytest.raises(vm.InvalidArgument, match=part):
            vm.Batch(**{**good, **change})


def test_tensors_of_the_wrong_type_are_refused_before_a_call():
    vm = package()
    operators = vm.operators
    for x, dtype, n, part in ((OnDevice(4, dtype=torch.int64), "i32", 4, "positions: of type torch.int64"), (OnDevice(4), "i32", 5, "want 5 values"),
                              (OnDevice(4, dtype=torch.bfloat16), "f32", 4, "of type torch.bfloat16"), (OnDevice(4, index=2), "i32", 4, "on cuda:2")):
        with pytest.raises(vm.InvalidArgument, match=part):
            operators._address("positions", x, dtype, n, 0)
    assert operators._address("positions", OnDevice(4), "i32", 4, 0) == 4096
    assert operators._address("lse", None, "f32", 4, 0) == 0 and operators._address("lse", 77, "f32", 4, 0) == 77


@pytest.mark.gpu
def test_tensors_give_what_their_addresses_give():
    from operator_refs import Paged, normal
    vm = package()
    rt = vm.Runtime.Create(0)
    scratch = vm.Scratch.Create(rt)
    p = Paged(rt, [3, 1], [20, 40], heads=2, q_heads=4, dim=64)
    r = vm.Rows.Of
    q = normal((4, 4, 64), "bf16", 1)
    out, lse = [torch.empty_like(q) for _ in range(2)], torch.zeros(2, 4, 4, device="cuda")
    batch = vm.Batch(2, p.start, p.length, p.table, p.table.shape[1], 4, 3)
    p.cache.Attend(p.batch, r(q), r(out[0]), scratch, lse=lse[0].data_ptr())
    p.cache.Attend(batch, r(q), r(out[1]), scratch, lse=lse[1])
    torch.cuda.synchronize()
    assert torch.equal(out[0], out[1]) and torch.equal(lse[0], lse[1]) and bool(lse[0].any())
    rope = vm.Rope.Create(rt, 64, 4, 0, "bf16", norm=True)
    pos, w = torch.arange(4, dtype=torch.int32, device="cuda"), 1 + 0.1 * normal((64,), "f32", 2)
    rope.Apply(4, pos.data_ptr(), r(q), None, r(out[0]), None, w.data_ptr())
    rope.Apply(4, pos, r(q), None, r(out[1]), None, w)
    dw = torch.zeros(2, 64, device="cuda")
    for i, args in enumerate(((pos.data_ptr(), w.data_ptr(), dw[0].data_ptr()), (pos, w, dw[1]))):
        rope.ApplyBackward(4, args[0], r(q), None, r(q), None, r(out[i].clone()), None, q_weight=args[1], dq_weight=args[2], scratch=scratch)
    torch.cuda.synchronize()
    assert torch.equal(out[0], out[1]) and torch.equal(dw[0], dw[1]) and bool(dw[0].any())
    for call in (lambda: rope.Apply(4, pos.long(), r(q), None, r(out[1]), None, w), lambda: rope.Apply(4, pos, r(q), None, r(out[1]), None, w.bfloat16()),
                 lambda: p.cache.Attend(batch, r(q), r(out[1]), scratch, lse=lse[1].double())):
        with pytest.raises(vm.InvalidArgument, match="of type"):
            call()
