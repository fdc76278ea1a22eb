"""Adapters (ovfq_project_adapters_dev) on whole numbers, where every sum is exact in fp32 in whatever order: the output is the
projection's plus the product, rounded once.

A product passes through 4 x shares chains (shares: 1 to 8 workgroups that divide the inputs) of three (bf16 adapters) or six (fp16,
fp32) MFMA accumulations for each 32 inputs, and how an MFMA rounds inside is the hardware's, so no order is assumed here. 16 inputs
of each rank have |A x| <= 2^18, the others A = 0: the magnitudes of every sum add up to at most 2^22. The bf16 parts that the kernel
divides x and A into are cut off, whole numbers of the whole's sign, and so their products' sums stay below that too. Each output
has three ranks with B = +-1 and the scale is 1/8: at most 3 * 2^22 < 2^24. The products of parts that the kernel leaves out for an
fp32 A (the second part with the third, the third with the third) are zeros: one factor has at most 8 bits, or both at most 16.
"""
import sys

import numpy as np
import pytest

from test_gpu_adapters import ELEMENT, make_weight

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
ov = pytest.importorskip("overfit_amd")

DEV = "cuda:0"
F32, F16, BF16 = ov.TYPE_F32, ov.TYPE_F16, ov.TYPE_BF16


def whole(gen, bits, *shape):
    """Whole numbers of `bits` bits and a sign, their top bit set (0 bits: +-1)."""
    top = 1 << max(bits - 1, 0)
    v = torch.randint(top, 2 * top, shape, generator=gen, device=DEV)
    return (v * (1 - 2 * torch.randint(0, 2, shape, generator=gen, device=DEV))).float()


def run(kind, k, n, rows, ranks, type_, x_bits, a_bits, own_rows=True):
    print("[case]", kind, k, n, rows, ranks, type_, x_bits, a_bits, own_rows, flush=True, file=sys.stderr)
    rng = np.random.default_rng(k + rows + n)
    gen = torch.Generator(device=DEV).manual_seed(k + rows + x_bits)
    w = make_weight(rng, kind, k, n)
    s = ov.AdapterSet(k, n, len(ranks) + 1, max(ranks), type_)
    x = whole(gen, x_bits, rows, k)
    slot = (torch.arange(rows, device=DEV) if own_rows else torch.arange(rows, device=DEV) * (len(ranks) + 1) // rows) % (len(ranks) + 1)
    slot = slot.to(torch.int32)  # (the last slot is empty)
    base = ov.project(w, x, rows=rows).view(rows, n)
    want = base.clone()
    for i, rank in enumerate(ranks):
        a, b = torch.zeros(rank, k, device=DEV), torch.zeros(n, rank, device=DEV)
        at = torch.rand(rank, k, generator=gen, device=DEV).topk(min(16, k), 1).indices
        at[:, 0] = k - 1 - torch.arange(rank, device=DEV) % k  # the last inputs too
        a.scatter_(1, at, whole(gen, a_bits, *at.shape))
        to = torch.rand(n, rank, generator=gen, device=DEV).topk(min(3, rank), 1).indices
        b.scatter_(1, to, whole(gen, 0, *to.shape))
        s.load(i, a.to(ELEMENT[type_]), b.to(ELEMENT[type_]), 0.125)
        mine = (slot == i).nonzero().squeeze(1)
        low = x[mine].double() @ a.double().t().contiguous()
        want[mine] += ((low @ b.double().t().contiguous()) * 0.125).float()
    got = ov.project_adapters([w], [s], x, slot, rows)[0].view(rows, n)
    wrong = (got != want).nonzero()
    assert not len(wrong), f"{len(wrong)} outputs, first {wrong[0].tolist()}: {got[tuple(wrong[0])]}, not {want[tuple(wrong[0])]}"


BITS = [(F32, 18, 0), (F32, 0, 18), (F32, 9, 9), (F32, 8, 10), (F16, 18, 0), (F16, 7, 11), (F16, 9, 9), (BF16, 18, 0), (BF16, 10, 8)]


# past 4096 rows no workgroup has a share of the inputs but the whole: the longest chains
@pytest.mark.parametrize("type_,x_bits,a_bits", BITS)
@pytest.mark.parametrize("kind,k,rows", [("q4k", 4096, 4112), ("q6k", 14336, 4112), ("q8", 2080, 4100)])
def test_whole_inputs_in_one_chain(kind, k, rows, type_, x_bits, a_bits):
    run(kind, k, 40, rows, (32, 7), type_, x_bits, a_bits, own_rows=False)


# the decode, split, panel and tiled kernels, rows of their own slots and prompts
@pytest.mark.parametrize("type_,x_bits,a_bits", BITS)
@pytest.mark.parametrize("kind,k,n,rows,ranks", [
    ("q4k", 4096, 300, 1, (16, 4)), ("q6k", 2304, 100, 5, (8, 20)), ("q8", 4096, 130, 3, (64,)), ("q4k", 14336, 64, 24, (40, 16, 3)),
    ("q8", 1056, 700, 45, (16, 5)), ("q4k", 2048, 2100, 150, (16, 64, 33)), ("q4k", 512, 5000, 600, (16, 3, 9, 12, 5, 16)),
])
def test_every_kernel_adds_the_exact_product(kind, k, n, rows, ranks, type_, x_bits, a_bits):
    for own_rows in (True, False):
        run(kind, k, n, rows, ranks, type_, x_bits, a_bits, own_rows)
