"""The adapters' first products as operands of the second: every bit of their fp32 value, in each output type."""
import pytest
import torch

from test_gpu_adapters import on_gpu

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16]


@pytest.fixture(scope="module")
def rt():
    from splosh_amd import runtime
    return runtime


def add(rt, x, a, b, out):
    """One adapter, every row its own: `x` [rows, inner], `a` [rank, inner], `b` [outputs, rank]."""
    got = out.cuda()
    adapters = (a[None].to(torch.bfloat16), b[None].to(torch.bfloat16), None, None)
    rt.add_adapters(got, x.to(torch.bfloat16).cuda(), on_gpu(rt, adapters), torch.zeros(len(x), dtype=torch.int32).cuda())
    return got.cpu()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,rank,inner,outputs", [(1, 2, 3, 5), (20, 8, 64, 64), (70, 40, 64, 96), (130, 16, 31, 64)])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_every_bit_reaches_the_output(rt, sign, rows, rank, inner, outputs, dtype):
    """1 + t0 - t1 with t0 = 1 + 2^-7 + 2^-9 + 2^-19 and t1 = 2^-9: 2^-19 past the middle of two bf16 numbers. (All of
    it is exact in fp32, whatever the order.)"""
    x, a, b = torch.zeros(rows, inner), torch.zeros(rank, inner), torch.zeros(outputs, rank)
    x[:, 0], x[:, 1], x[:, 2] = 1.0, 2.0 ** -9, 2.0 ** -19
    a[0, 0], a[0, 1], a[0, 2], a[1, 1] = 1.0 + 2.0 ** -7, 1.0, 1.0, 1.0
    b[:, 0], b[:, 1] = sign, -sign
    got = add(rt, x, a, b, torch.full((rows, outputs), sign, dtype=dtype))
    want = 2.0 + 2.0 ** -6 if dtype == torch.bfloat16 else 2.0 + 2.0 ** -7 + 2.0 ** -19
    assert (got.float() == sign * want).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_products_at_the_end_of_fp32(rt, sign, dtype):
    """t = 2^127 (1 + 0.99609375 + 2^-11), finite but nearer to 2^128 than to any bf16 number: 2^-126 of it is 4 - 2^-7 + 2^-10."""
    x, a, b = torch.zeros(3, 8), torch.zeros(4, 8), torch.zeros(16, 4)
    x[:, :3] = 2.0 ** 64
    a[0, 0], a[0, 1], a[0, 2] = sign * 2.0 ** 63, sign * 0.99609375 * 2.0 ** 63, sign * 2.0 ** 52
    b[:, 0] = 2.0 ** -126
    got = add(rt, x, a, b, torch.zeros(3, 16, dtype=dtype))
    want = torch.tensor(2.0 * (1.0 + 0.99609375 + 2.0 ** -11)).to(dtype)
    assert (got == sign * want).all()


def test_the_most_rows(rt):
    """2^21 rows, the entry points' limit: 32768 chunks."""
    from adapter_check import check
    from test_gpu_adapters import host_case, slots_of
    rows = 1 << 21
    x, adapters, out = host_case(rows, 8, 16, 3, 3, torch.bfloat16, 43)
    slots = slots_of(rows, 3, 43)
    got = rt.add_adapters(out.cuda(), x.cuda(), on_gpu(rt, adapters), slots.cuda())
    pick = list(range(0, 200)) + list(range(rows // 2 - 100, rows // 2 + 100)) + list(range(rows - 200, rows))
    check(got[pick], out[pick], x[pick], adapters, slots[pick])
    idle = (slots < 0) | (slots >= 3)
    assert torch.equal(got.cpu()[idle].view(torch.int16), out[idle].view(torch.int16))
