"""The 4-bit paged cache's layout and quantiser in plain torch, for the tests: a block of 64 tokens holds the codes of all
tokens (head dim / 2 bytes each), then their F16 scales (head dim / 32 each); word w of a token (8 codes) stands at place
(w % 4) * (head dim / 32) + w / 4."""
import torch

PAGE = 64


def places(dim):
    """Byte and shift of every element's code within its token's codes."""
    e = torch.arange(dim)
    word = e // 8
    return ((word % 4) * (dim // 32) + word // 4) * 4 + e % 8 // 2, 4 * (e % 2)


def decode(pool):
    """(values f64, scales f64 per element, codes) [...][64][head dim] of a uint8 pool [...][64][9 / 16 head dim]."""
    dim = pool.shape[-1] // 9 * 16
    flat = pool.flatten(-2).contiguous()
    byte, shift = (t.to(pool.device) for t in places(dim))
    rows = flat[..., :PAGE * dim // 2].unflatten(-1, (PAGE, dim // 2))
    code = (rows[..., byte].long() >> shift) & 15
    scale = flat[..., PAGE * dim // 2:].contiguous().view(torch.float16).unflatten(-1, (PAGE, dim // 32))
    scale = scale.double().repeat_interleave(32, -1)
    return scale * (code - 8).double(), scale, code


def quantise(x):
    """(codes [...][dim], scales f16 [...][dim / 32]) of values [...][dim], step by step in f32."""
    g = x.float().unflatten(-1, (-1, 32))
    big = g.abs().amax(-1)
    m = torch.where((g == -big[..., None]).any(-1), -big, big)
    t = torch.where(torch.isfinite(g).all(-1), (m / -8.0).clamp(-2720.0, 2720.0), float("nan"))
    scale = t.to(torch.bfloat16).to(torch.float16)
    s = scale.float()[..., None]
    inv = torch.where(s != 0, 1.0 / s, 0.0)
    code = torch.floor(g * inv + 8.5).nan_to_num(0.0).clamp(0.0, 15.0)
    return code.to(torch.uint8).flatten(-2), scale


def encode(x):
    """uint8 pool [...][64][9 / 16 dim] of values [...][64][dim]."""
    dim = x.shape[-1]
    code, scale = quantise(x)
    byte, shift = places(dim)
    rows = torch.zeros(*x.shape[:-1], dim // 2, dtype=torch.uint8, device=x.device)
    for low in (0, 1):
        at = (shift == 4 * low).nonzero()[:, 0].to(x.device)
        rows[..., byte.to(x.device)[at]] |= code[..., at] << (4 * low)
    flat = torch.cat((rows.flatten(-2), scale.contiguous().view(torch.uint8).flatten(-2)), -1)
    return flat.unflatten(-1, (PAGE, 9 * dim // 16)).contiguous()
