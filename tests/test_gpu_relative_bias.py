"""Relative-position bias by buckets (ops.relative_bias): the forward copies
table entries, so it equals the definition exactly; the table's gradient is a sum of fp32
terms, at most 512 of them in a chain (a thread's run, then the partial rows),
so within 512 u of the sum of their magnitudes, u = 2^-24, before it is rounded."""

import pytest
import torch

from boltz_lumi_amd import ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def bucket_table(side, exact, top, far):
    """Buckets of the distances 0 .. far of one direction, from the definition in whole numbers."""
    def one(n):
        if n < exact:
            return n
        return exact + max(k for k in range(side - exact) if n ** (side - exact) >= exact ** (side - exact - k) * top ** k)
    return torch.tensor([one(n) for n in range(far + 1)])


def buckets_of(q_pos, k_pos, buckets, exact, top, bidirectional):
    side = buckets // 2 if bidirectional else buckets
    far = max(exact, top) + 2
    table = bucket_table(side, exact, top, far).to(q_pos.device)
    d = k_pos[..., None, :].long() - q_pos[..., :, None].long()
    if bidirectional:
        return table[d.abs().clamp(max=far)] + side * (d > 0)
    return table[(-d).clamp(0, far)]


CASES = [  # batch, m, n, heads, buckets, exact, max distance, bidirectional, dtype, gaps
    (None, 1, 1, 1, 2, 1, 128, False, torch.float32, False),
    (None, 1, 1531, 16, 32, 16, 128, False, torch.bfloat16, False),
    (None, 130, 257, 3, 32, 8, 128, True, torch.float32, False),
    (None, 65, 129, 5, 66, 32, 32, True, torch.bfloat16, True),
    (2, 77, 31, 4, 128, 20, 5000, True, torch.float32, True),
    (3, 9, 2049, 2, 256, 64, 300, True, torch.bfloat16, True),
    (1, 2100, 5, 16, 64, 63, 64, False, torch.float32, True),
    (None, 700, 801, 12, 32, 4, 9, False, torch.bfloat16, False),
]


def make(case, gpu):
    batch, m, n, heads, buckets, _, _, _, dtype, gaps = case
    g = torch.Generator(device=gpu).manual_seed(m + n)
    table = torch.randn(buckets, heads, generator=g, device=gpu).to(dtype)

    def positions(t, lead):
        if not gaps:
            return torch.arange(t, device=gpu).expand(*lead, t)
        return torch.randint(-6000, 6000, (*lead, t), generator=g, device=gpu)

    lead = () if batch is None else (batch,)
    return table, positions(m, lead), positions(n, ()), g  # the keys' positions are shared by the batch


@pytest.mark.parametrize("case", CASES)
def test_forward_and_gradient(gpu, case):
    print(f"relative_bias {case}", flush=True)
    batch, m, n, heads, buckets, exact, top, bidirectional, dtype, _ = case
    table, q_pos, k_pos, g = make(case, gpu)
    table.requires_grad_()
    bias = ops.relative_bias(table, q_pos, k_pos, exact=exact, max_distance=top, bidirectional=bidirectional)
    index = buckets_of(q_pos, k_pos, buckets, exact, top, bidirectional)
    want = table.detach()[index].movedim(-1, -3)
    assert bias.is_contiguous() and torch.equal(bias.detach(), want)
    dbias = torch.randn(bias.shape, generator=g, device=gpu).to(dtype)
    dtable, = torch.autograd.grad(bias, table, dbias)
    flat = dbias.double().movedim(-3, -1).reshape(-1, heads)
    shape = (buckets, heads)
    sums = torch.zeros(shape, device=gpu, dtype=torch.float64).index_add_(0, index.flatten(), flat)
    size = torch.zeros(shape, device=gpu, dtype=torch.float64).index_add_(0, index.flatten(), flat.abs())
    err = (dtable.double() - sums).abs() - 512 * U * size - torch.finfo(dtype).eps / 2 * sums.abs()
    assert bool((err <= 1e-30).all()), err.max().item()
    with torch.no_grad():
        half = ops.relative_bias(table, q_pos.int(), k_pos.int(), exact=exact, max_distance=top,
                                 bidirectional=bidirectional)
    assert torch.equal(half, bias.detach())


def test_far_positions(gpu):
    """64-bit positions whose distances pass 32 bits fall into the last buckets."""
    table = torch.arange(64, device=gpu, dtype=torch.float32).view(32, 2)
    q_pos = torch.tensor([0, 1 << 61, -(1 << 61)], device=gpu)
    k_pos = torch.tensor([0, (1 << 61) + 1, -(1 << 40), 1 << 33], device=gpu)
    bias = ops.relative_bias(table, q_pos, k_pos)
    index = torch.tensor([[0, 31, 15, 31], [15, 17, 15, 15], [31, 31, 31, 31]], device=gpu)
    assert torch.equal(bias, table[index].movedim(-1, 0))


def test_large_plane(gpu):
    """More than 2^31 elements: offsets in 64 bits (bf16, 4.5 GB)."""
    heads, m, n = 9, 16001, 16003
    table = torch.randn(32, heads, device=gpu, dtype=torch.bfloat16)
    q_pos, k_pos = torch.arange(m, device=gpu), torch.arange(n, device=gpu)
    bias = ops.relative_bias(table, q_pos, k_pos)
    index = buckets_of(q_pos[-3:], k_pos, 32, 8, 128, True)
    assert torch.equal(bias[:, -3:], table[index].movedim(-1, 0))
    dbias = torch.zeros_like(bias)
    dbias[-1, -1, -1] = 1.5
    dbias[-1, -1, 0] = 0.25
    table.requires_grad_()
    dtable, = torch.autograd.grad(ops.relative_bias(table, q_pos, k_pos), table, dbias)
    want = torch.zeros_like(table)
    want[buckets_of(q_pos[-1:], k_pos[-1:], 32, 8, 128, True)[0, 0], -1] = 1.5
    want[15, -1] = 0.25
    assert torch.equal(dtable, want)


def test_empty_and_repeated(gpu):
    table = torch.randn(32, 3, device=gpu, requires_grad=True)
    none = torch.arange(0, device=gpu)
    some = torch.arange(5, device=gpu)
    for q_pos, k_pos, shape in ((none, some, (3, 0, 5)), (some, none, (3, 5, 0)),
                                (some.expand(0, 5), some, (0, 3, 5, 5))):
        bias = ops.relative_bias(table, q_pos, k_pos)
        assert bias.shape == shape
        assert not torch.autograd.grad(bias.sum() + 0 * table.sum(), table)[0].any()
    bias = ops.relative_bias(table, torch.arange(300, device=gpu), torch.arange(500, device=gpu))
    dbias = torch.randn_like(bias)
    first = torch.autograd.grad(bias, table, dbias, retain_graph=True)[0]
    for _ in range(3):
        assert torch.equal(first, torch.autograd.grad(bias, table, dbias, retain_graph=True)[0])
    # an expanded (stride 0) gradient, and the linear map's differences
    total = torch.autograd.grad(bias.sum(), table, retain_graph=True)[0]
    v = torch.randn_like(table)
    with torch.no_grad():
        moved = ops.relative_bias(table + v, torch.arange(300, device=gpu), torch.arange(500, device=gpu))
    change, want = (moved.double() - bias.double()).sum().item(), (total.double() * v).sum().item()
    size = bias.double().abs().sum().item() + moved.double().abs().sum().item()
    assert abs(change - want) <= 4 * U * size  # each entry of table + v and its difference rounds once


def test_refusals(gpu):
    table, pos = torch.zeros(32, 4, device=gpu), torch.arange(6, device=gpu)
    good = dict(table=table, q_pos=pos, k_pos=pos)
    for change, text in [
        ({"table": table[0]}, "table"), ({"table": table.half()}, "dtype"), ({"table": table[:31]}, "even"),
        ({"table": table[:2]}, "two buckets"), ({"table": torch.zeros(258, 4, device=gpu)}, "256"),
        ({"q_pos": pos.float()}, "int32 or int64"), ({"q_pos": pos.int()}, "share"),
        ({"q_pos": pos.view(1, 1, 6)}, "positions"), ({"q_pos": pos.expand(2, 6), "k_pos": pos.expand(3, 6)}, "shape"),
        ({"exact": 16}, "exact"), ({"exact": 0}, "exact"), ({"max_distance": 8}, "max_distance"),
        ({"max_distance": 1 << 31}, "max_distance"), ({"table": table.cpu()}, "CUDA"), ({"k_pos": pos.cpu()}, "CUDA"),
    ]:
        with pytest.raises(RuntimeError, match=text):
            ops.relative_bias(**{**good, **change})
