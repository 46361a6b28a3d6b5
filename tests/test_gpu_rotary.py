"""Rotary positions on the GPU against the float64 restatement, forward and backward.

Bars, on the largest error over the largest value.  A rotated value is a c - b s in float32, two products and a difference,
each rounded, with the table's cos and sin as given: at most 3 x 2^-24 (|a| + |b|), |a| + |b| up to twice the largest
value; and the rounding to the dtype, at most 2^-8 (bf16), 2^-11 (f16) or 2^-24 of the value."""
import pytest
import torch

from _parity import check
from macai.layer import rotary, rotary_table
from oracle import attention as A

pytestmark = pytest.mark.gpu
ROUND = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -9, torch.float16: 2.0 ** -11}


def _err(x, ref):
    return float((x.detach().double().cpu() - ref).abs().max() / ref.abs().max().clamp(min=1e-30))


def _bar(dtype):
    return 2 * ROUND[dtype] + 8 * 2.0 ** -24      # max |y| may be under max (|a| + |b|) by up to sqrt 2


def _case(shape, Hq, Hk, D, width, dtype, seed, positions=64):
    gen = torch.Generator().manual_seed(seed)
    q, k = torch.randn(*shape, Hq, D, generator=gen).to(dtype), torch.randn(*shape, Hk, D, generator=gen).to(dtype)
    return q, k, rotary_table(width, positions, 500.0, device="cuda"), gen


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape,Hq,Hk,D,width", [((1, 1), 1, 1, 16, 16), ((2, 5), 3, 1, 64, 16), ((1, 33), 16, 2, 256, 64),
                                                 ((3, 7), 5, 5, 80, 48), ((9,), 4, 2, 128, 128), ((2, 3), 2, 0, 96, 32)])
def test_forward_backward(shape, Hq, Hk, D, width, interleaved, dtype):
    q, k, table, gen = _case(shape, Hq, Hk, D, width, dtype, 1)
    pos = torch.randint(0, 64, shape, generator=gen, dtype=torch.int32)
    dq, dk = torch.randn(q.shape, generator=gen).to(dtype), torch.randn(k.shape, generator=gen).to(dtype)
    lq, lk = q.cuda().requires_grad_(True), k.cuda().requires_grad_(True)
    qo, ko = rotary(lq, lk, table, pos.cuda(), interleaved)
    gq, gk = torch.autograd.grad([qo, ko], [lq, lk], [dq.cuda(), dk.cuda()])
    assert qo.dtype == gq.dtype == dtype and qo.shape == q.shape and gk.shape == k.shape
    t = table.cpu()
    errs = {"q": _err(qo, A.rotate(q, t, pos, interleaved)), "dq": _err(gq, A.rotate(dq, t, pos, interleaved, True))}
    if Hk:
        errs["k"] = _err(ko, A.rotate(k, t, pos, interleaved))
        errs["dk"] = _err(gk, A.rotate(dk, t, pos, interleaved, True))
    check(errs, _bar(dtype))


@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient_is_the_difference_quotient(interleaved):
    """The rotation is linear: (f(x + e) - f(x - e)) . g / 2 = e . df(g), up to float32 rounding of the sums."""
    q, k, table, gen = _case((1, 21), 3, 2, 64, 32, torch.float32, 2)
    pos = torch.arange(21).cuda()
    eq, ek, gq, gk = (torch.randn(x.shape, generator=gen).cuda() for x in (q, k, q, k))
    q, k = q.cuda().requires_grad_(True), k.cuda().requires_grad_(True)
    dq, dk = torch.autograd.grad(rotary(q, k, table, pos, interleaved), [q, k], [gq, gk])
    with torch.no_grad():
        hi, lo = rotary(q + eq, k + ek, table, pos, interleaved), rotary(q - eq, k - ek, table, pos, interleaved)
    quotient = sum(((a - b).double() * g.double()).sum() for a, b, g in zip(hi, lo, (gq, gk))) / 2
    slope = (dq.double() * eq.double()).sum() + (dk.double() * ek.double()).sum()
    # n independent terms of size about 1, each with a few roundings of 2^-24
    assert abs(float(quotient - slope)) < 8 * 2.0 ** -24 * (q.numel() + k.numel()) ** 0.5 * 4


@pytest.mark.parametrize("wide", [torch.int32, torch.int64])
def test_strides_shared_positions_and_gradients_of_one(wide):
    """Slices of a projection's output and a transposed layout are read where they are; positions [T] serve every row of a
    batch; a broadcast gradient and one that is missing."""
    gen = torch.Generator().manual_seed(3)
    table = rotary_table(64, 40, device="cuda")
    qkv = torch.randn(2, 11, 8, 64, generator=gen).to(torch.bfloat16)
    pos = torch.arange(7, 18, dtype=wide)
    dev = qkv.cuda()
    qo, ko = rotary(dev[:, :, :4], dev[:, :, 4:6], table, pos.cuda())
    check({"q": _err(qo, A.rotate(qkv[:, :, :4], table.cpu(), pos.expand(2, 11))),
           "k": _err(ko, A.rotate(qkv[:, :, 4:6], table.cpu(), pos.expand(2, 11)))}, _bar(torch.bfloat16))
    t = dev.transpose(1, 2).contiguous().transpose(1, 2)          # [B, H, T, D] in memory
    q2, _ = rotary(t[:, :, :4], t[:, :, 4:6], table, pos.cuda())
    assert torch.equal(q2, qo)
    odd = torch.empty(dev.numel() + 1, dtype=dev.dtype, device="cuda")[1:].view(dev.shape).copy_(dev)   # misaligned
    assert torch.equal(rotary(odd[:, :, :4], odd[:, :, 4:6], table, pos.cuda())[0], qo)
    leaf = dev[:, :, :4].clone().requires_grad_(True)
    q3, _ = rotary(leaf, dev[:, :, 4:6], table, pos.cuda())
    g = torch.ones(1, 1, 1, 64, dtype=torch.bfloat16, device="cuda").expand(q3.shape)
    (dq,) = torch.autograd.grad(q3, leaf, g)
    check({"dq": _err(dq, A.rotate(g.cpu(), table.cpu(), pos.expand(2, 11), back=True))}, _bar(torch.bfloat16))


def test_positions_outside_of_the_table_are_nan():
    q, k, table, _ = _case((1, 4), 2, 1, 64, 32, torch.bfloat16, 4, positions=8)
    qo, ko = rotary(q.cuda(), k.cuda(), table, torch.tensor([0, 8, -1, 7], device="cuda"))
    for x, y in ((q, qo.cpu()), (k, ko.cpu())):
        assert torch.isnan(y[0, 1:3, :, :32]).all() and not torch.isnan(y[0, 0::3]).any()
        assert torch.equal(y[..., 32:], x[..., 32:])


def test_no_tokens_and_another_stream():
    table = rotary_table(16, 4, device="cuda")
    q = torch.empty(2, 0, 3, 16, device="cuda", requires_grad=True)
    qo, ko = rotary(q, torch.empty(2, 0, 1, 16, device="cuda"), table, torch.empty(0, dtype=torch.int64, device="cuda"))
    assert qo.shape == (2, 0, 3, 16) and ko.shape == (2, 0, 1, 16)
    assert torch.autograd.grad(qo.sum(), q)[0].shape == q.shape
    q, k, table, _ = _case((1, 500), 4, 2, 64, 64, torch.float32, 5, positions=500)
    q, k, pos = q.cuda(), k.cuda(), torch.arange(500, device="cuda")
    want = rotary(q, k, table, pos)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = rotary(q, k, table, pos)
    s.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
