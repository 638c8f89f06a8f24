"""The MXFP4 format of a cache from its definition, in 64 bits, and caches of it."""
import math

import torch

from tests.attention_util import Step

VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
EXPONENTS = {torch.float16: (-23, 13), torch.bfloat16: (-125, 125)}


def _power(e):
    """2^e for whole numbers from -300 to 300, exactly."""
    return torch.tensor([2.0 ** i for i in range(-300, 301)], dtype=torch.float64, device=e.device)[e.long() + 300]


def widths(dim):
    """Bytes of a row of codes, and of its scales."""
    return 16 * math.ceil(dim / 32), 2 if dim <= 64 else 4 if dim <= 128 else 8


def encode(x, dtype=None):
    """(codes, scales) of rows [..., dim]: scales of the groups there are."""
    low, high = EXPONENTS[dtype or x.dtype]
    x = torch.nn.functional.pad(x.double(), (0, -x.shape[-1] % 32)).unflatten(-1, (-1, 32))
    fine = x.isfinite().all(-1)
    x = torch.where(fine[..., None], x, 0.0)
    most = x.abs().amax(-1)
    power = torch.frexp(most)[1] - 1                                     # 2^power <= most < 2^(power + 1)
    e = (power - 2 + (most >= 1.75 * _power(power))).clamp(low, high)
    e = torch.where(most == 0, low, e)
    size = x.abs() * _power(-e[..., None])
    values = torch.tensor(VALUES, dtype=torch.float64, device=x.device)
    off = (size[..., None] - values).abs()
    nearest = off == off.amin(-1, keepdim=True)
    # of two codes that are as near, the even one
    odd = torch.arange(8, device=x.device) % 2 == 1
    code = torch.where(nearest & ~(odd & (nearest.sum(-1, keepdim=True) > 1)), 1, 0).argmax(-1)
    code = torch.where(fine[..., None], code + 8 * torch.signbit(x), 0).flatten(-2).to(torch.uint8)
    return code[..., ::2] + 16 * code[..., 1::2], torch.where(fine, e + 127, 255).to(torch.uint8)


def decode(codes, scales, dim):
    """What rows of bytes stand for, in 64 bits."""
    values = torch.tensor(VALUES + tuple(-v for v in VALUES), dtype=torch.float64, device=codes.device)
    rows = torch.stack((values[(codes % 16).long()], values[(codes // 16).long()]), -1).flatten(-2)
    scales = scales[..., :codes.shape[-1] // 16]
    power = torch.where(scales == 255, math.nan, _power(scales.int() - 127))
    return (rows.unflatten(-1, (-1, 32)) * power[..., None]).flatten(-2)[..., :dim]


def empty(blocks, block_size, heads, dim, layout="head", device="cuda", code=0x7A, scale=255):
    """Keys and values of a cache as (codes, scales) each, whose rows stand for NaN."""
    from autogptq.tvm_amd.attention import Mxfp4

    made = []
    for n, fill in zip(widths(dim), (code, scale)):
        shape = (2, blocks, block_size, heads, n) if layout == "token" else (2, blocks, heads, block_size, n)
        both = torch.full(shape, fill, dtype=torch.uint8, device=device)
        made.append(both if layout == "token" else both.transpose(2, 3))
    return Mxfp4(made[0][0], made[1][0]), Mxfp4(made[0][1], made[1][1])


class MxStep(Step):
    """A ``Step`` whose cache is held in MXFP4: what the oracle sees are the values that the codes stand for.  (What no token may read
    is NaN here, too.)"""

    def __init__(self, *args, **more):
        super().__init__(*args, **more)
        self.quantise()

    def quantise(self):
        from autogptq.tvm_amd.attention import Mxfp4

        packed = []
        for cache in (self.k_cache, self.v_cache):
            codes, scales = encode(cache)
            n = widths(self.dim)[1]
            scales = torch.nn.functional.pad(scales, (0, n - scales.shape[-1]), value=255)
            # in the memory order of the cache
            heads_first = cache.stride(2) > cache.stride(1)
            order = (lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)) if heads_first else (lambda t: t.contiguous())
            packed.append(Mxfp4(order(codes), order(scales)))
        self.k_cache, self.v_cache = packed
        self.k, self.v = ([decode(*encode(x), self.dim) for x in rows] for rows in (self.k, self.v))
