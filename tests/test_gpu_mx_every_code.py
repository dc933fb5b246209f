"""Every E2M1 code under every scale byte, as a pool of another program may hold them: read
back as rows, and as keys and values of attention."""

import math

import pytest
import torch

from mx_reference import VALUES, decode
from neptune_hip import ops

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")


def _pools(D):
    """256 pages of 16 places: block 0 of page e's place 0 is all codes, twice, under byte
    e; the other blocks are 1 under 2^0."""
    codes = torch.full((256, 1, 16, D // 2), 0x22, dtype=torch.uint8)
    byte = torch.full((256, 1, 16, D // 32), 127, dtype=torch.uint8)
    c = torch.arange(32, dtype=torch.uint8) % 16
    codes[:, 0, 0, :16] = c[0::2] | c[1::2] << 4
    byte[:, 0, 0, 0] = torch.arange(256).to(torch.uint8)
    want = decode(codes[:, 0, 0], byte[:, 0, 0])
    two = torch.exp2(torch.arange(256).double() - 127)
    assert torch.equal(want[:255, :8], (VALUES * two[:, None])[:255])  # (code 8 is -0)
    table = torch.arange(256, dtype=torch.int32)[:, None]
    lens = torch.ones(256, dtype=torch.int32)
    return want, (codes.cuda(), byte.cuda()), table.cuda(), lens.cuda()


def _same(got, want, tiny):
    """Equal, but that products below `tiny` may be 0."""
    got = got.double()
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    zero = (want.abs() < tiny) & (got == 0)
    ok = (got == want) | zero | nan
    assert ok.all(), (got[~ok][:8], want[~ok][:8])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_read(dtype, D):
    want, (codes, byte), table, lens = _pools(D)
    k, v = ops.kv_read_paged(codes, codes, table, lens, dtype=dtype, k_scales=byte, v_scales=byte)
    torch.cuda.synchronize()
    # (past the type's range: infinite; f16 below 2^-14: to steps of 2^-24)
    rounded = want.to(F32).to(dtype).double()
    for x in (k, v):
        _same(x[:, 0].cpu(), rounded, 2.0**-24 if dtype == F16 else 2.0**-126)


@pytest.mark.parametrize("window", [None, 1])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_values(dtype, D, window):
    """One key a sequence: the output is its value, in the queries' type."""
    want, (codes, byte), table, lens = _pools(D)
    ones = torch.full_like(codes, 0x22), torch.full_like(byte, 127)
    q = torch.randn(256, 2, D, generator=torch.Generator().manual_seed(1)).to(dtype)
    o = ops.attention_paged(q.cuda(), ones[0], codes, table, lens, window=window,
                            max_seq_len=16, k_scales=ones[1], v_scales=byte)
    torch.cuda.synchronize()
    rounded = want.to(F32).to(dtype).double()
    rounded[torch.isinf(rounded)] = math.inf  # checked by magnitude below
    got = o.cpu()
    for h in range(2):
        x = got[:, h].double()
        inf = torch.isinf(rounded)
        assert torch.isinf(x[inf]).all()
        assert torch.equal(torch.sign(x[inf]), torch.sign(want[inf]))
        _same(x.where(~inf, 0.0), rounded.where(~inf, 0.0),
              2.0**-24 if dtype == F16 else 2.0**-126)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_keys(dtype, D):
    """One key a sequence, queries of one element each: the log-sum-exp is the product."""
    want, (codes, byte), table, lens = _pools(D)
    ones = torch.full_like(codes, 0x22), torch.full_like(byte, 127)
    q = torch.zeros(256, 16, D, dtype=dtype)
    q[:, torch.arange(16), torch.arange(16)] = 1.0
    _, lse = ops.attention_paged(q.cuda(), codes, ones[0], table, lens, return_lse=True, scale=1.0,
                                 max_seq_len=16, k_scales=byte, v_scales=ones[1])
    torch.cuda.synchronize()
    k = want.to(F32).to(dtype).double()
    s = (q.double() * k[:, None]).sum(-1)  # (0 times an infinity or NaN is NaN, there too)
    got = lse.cpu().double()
    plain = s.abs() < 2.0**120
    assert torch.isnan(got[torch.isnan(s)]).all()
    tiny = 2.0**-24 if dtype == F16 else 2.0**-126
    # log2(e) and back: three roundings of 2^-24, and 2^-24 of l's logarithm, which is 0
    off = (got - s).abs()[plain]
    assert (off <= 2.0**-22 * s.abs()[plain] + tiny).all()
