"""Codes of stored 16-bit rows next to a half: every pair of significands and every power of two between them that changes a code.

127 x / a of 16-bit x and a is a half, or no nearer to one than 2^-18.9 of it (fp16: a = 2047, x = 1910; bf16 2^-16.0: a = 255, x = 254)."""
import pytest
import torch

from gpu_util import DEV
from test_gpu_int8 import ops  # noqa: F401

pytestmark = pytest.mark.gpu


def rows_and_codes(bits, lower):
    """A row per significand a; its values all s 2^-e.  Codes by integers: rint(127 s / (a 2^e)), halves to even."""
    sig = torch.arange(1 << (bits - 1), 1 << bits)
    e = torch.arange(0, 11)
    s, shift = sig.repeat(len(e)), e.repeat_interleave(len(sig))
    a = sig[:, None]
    num, den = 254 * s[None, :], a << shift[None, :]          # twice the quotient
    whole, left = num // (2 * den), num % (2 * den)
    codes = whole + ((left > den) | ((left == den) & (whole % 2 == 1))).long()
    x = (s.double() * 2.0 ** -shift.double())[None, :].expand(len(sig), -1).clone()
    inside = x <= a.double()
    x, codes = torch.where(inside, x, 0.0), torch.where(inside, codes, 0)
    x[:, 1::2] *= -1
    codes[:, 1::2] *= -1
    scale = 2.0 ** -lower
    return torch.cat([a.double() * scale, x * scale], 1), torch.cat([torch.full_like(a, 127), codes], 1)


def test_the_nearest_quotients():
    for a, x, e, half, bound in [(2047, 1910, 0, 118.5, 18.89), (2031, 2047, 8, 0.5, 17.99), (255, 254, 0, 126.5, 15.98), (253, 255, 8, 0.5, 14.99)]:
        q = 127 * x / (a * 2 ** e)
        assert 0 < abs(q - half) / half < 2.0 ** -(bound - 0.02) and abs(q - half) / half > 2.0 ** -bound


@pytest.mark.parametrize("dt,bits,lower", [(torch.float16, 11, 0), (torch.float16, 11, 8), (torch.bfloat16, 8, 0), (torch.bfloat16, 8, 30), (torch.bfloat16, 8, -100)])
def test_every_pair_of_significands(ops, dt, bits, lower):  # noqa: F811
    x, codes = rows_and_codes(bits, lower)
    v = x.to(dt)
    assert torch.equal(v.double(), x) or dt == torch.float16 and lower      # fp16: some of the smallest are subnormal
    if not torch.equal(v.double(), x):
        codes = torch.where(v.double() == x, codes, 0)
        v = torch.where(v.double() == x, v, 0)
    for pad in (0, -v.shape[1] % 8):                           # element by element; sixteen bytes at a time
        row = torch.nn.functional.pad(v, (0, pad))
        q, s = ops.quantize_int8(row.to(DEV))
        assert torch.equal(q.cpu()[:, :codes.shape[1]].long(), codes)
        a = row[:, 0].float()
        assert torch.equal(s.cpu(), a / torch.full_like(a, 127.0))
