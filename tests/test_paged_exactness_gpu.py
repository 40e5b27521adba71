"""What the paged kernels may lose to rounding, where it shows: in differences of nearly equal numbers."""
import pytest
import torch

from dart_pytorch_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd,heads,page", [(64, 1, 16), (128, 4, 16), (64, 16, 8), (128, 12, 1), (256, 2, 32), (33, 1, 4)])
def test_weights_have_all_their_bits(hd, heads, page):
    """Two keys of weights 1 and exp(-x) with values 1 and -1 leave tanh(x / 2), a few 2^-18 of either.

    exp2 is off by 2^-22 of its result at most, a sum of 32 bits that truncates by 2^-23 for each of the three parts of a weight, and the
    quotient by less; half of that reaches the output, which is rounded to 8 bits.  Weights of 16 bits would be off by up to 2^-18."""
    x = torch.arange(1, 128, 2, device="cuda", dtype=torch.float32) * 2.0 ** -18       # (exact in bf16; 16 bits would end at 2^-17)
    rows = len(x)
    pages = -(-2 // page)
    k, v = (torch.zeros(rows * pages, 1, page, hd, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    table = torch.arange(rows * pages, dtype=torch.int32, device="cuda").view(rows, pages)
    second = (table[:, -1].long(), 0, 1 % page)
    k[second + (0,)] = -x.bfloat16()
    v[table[:, 0].long(), 0, 0] = 1.0
    v[second] = -1.0
    q = torch.zeros(rows, heads, hd, dtype=torch.bfloat16, device="cuda")
    q[..., 0] = 1.0
    got = ops.paged_attention(q, k, v, table, torch.full((rows,), 2, dtype=torch.int32, device="cuda"), scale=1.0).double()
    want = torch.tanh(x.double() / 2)[:, None, None]
    assert bool(((got - want).abs() <= want * 2.0 ** -8 + 5 * 2.0 ** -24).all())


@pytest.mark.parametrize("hd,heads", [(64, 1), (128, 4), (128, 16), (64, 9), (256, 2)])
def test_long_sums_do_not_drift(hd, heads):
    """Half of the keys again, with values of the other sign: what is summed up first goes down to zero, one row a warp.

    A running sum of at most 1.5 takes 512 roundings or fewer each way, 2^-24 of it: at worst an output is off by 1024 * 1.5 * 2^-24, and
    rounded to nearest there is no sign to it, so the mean of n of them stays below 7 / sqrt(n) of that.  Values of a sum that truncates shrink in both
    halves, all to one side: by 8e-6."""
    g = torch.Generator(device="cuda").manual_seed(hd + heads)
    n, page, rows = 4096, 16, 1184
    k = torch.randn(n // page, 1, page, hd, generator=g, device="cuda").bfloat16()
    v = (torch.rand(n // page, 1, page, hd, generator=g, device="cuda") + 0.5).bfloat16()
    table = torch.arange(2 * n // page, device="cuda", dtype=torch.int32).expand(rows, -1).contiguous()
    q = torch.randn(rows, heads, hd, generator=g, device="cuda").bfloat16()
    o = ops.paged_attention(q, torch.cat([k, k]), torch.cat([v, -v]), table, torch.full((rows,), 2 * n, device="cuda", dtype=torch.int32)).double()
    worst = 1024 * 1.5 * 2.0 ** -24
    assert float(o.abs().max()) <= worst and abs(float(o.mean())) <= 7 * worst / o.numel() ** 0.5


@pytest.mark.parametrize("rotary,hd", [(64, 64), (128, 128), (32, 80)])
@pytest.mark.parametrize("base", [10000.0, 500000.0])
def test_sine_and_cosine_are_rounded_once(rotary, hd, base):
    """Pairs (1, 0) and (0, 1) become the cosine and the sine themselves: half a step from the angle's in 64 bits, which a position p has to
    2^-50 p (three roundings of it, and exp2)."""
    positions = [1, 2, 3, 7, 100, 777, 4095, 30011, 131071, 10 ** 6, 2 ** 31 - 1]
    tokens, half = len(positions), rotary // 2
    p = torch.tensor(positions, dtype=torch.float64)[:, None]
    angle = p * base ** (-2.0 * torch.arange(half, dtype=torch.float64) / rotary)
    cos, sin = torch.cos(angle), torch.sin(angle)
    k, v = (torch.empty(1, 1, 2 ** 20, hd, device="cuda") for _ in range(2))            # one page in all places
    table = torch.zeros(1, 2 ** 11, dtype=torch.int32, device="cuda")
    qkv = torch.zeros(tokens, 4, hd, device="cuda")
    qkv[:, 0, :half] = 1.0
    qkv[:, 1, half:rotary] = 1.0
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    q = ops.paged_append(qkv.view(tokens, -1), k, v, table, ints(positions), 2, rows=ints([0] * tokens), rotary_dim=rotary,
                         rope_base=base).double().cpu()
    for got, want in ((q[:, 0, :half], cos), (q[:, 0, half:rotary], sin), (q[:, 1, :half], -sin), (q[:, 1, half:rotary], cos)):
        assert bool(((got - want).abs() <= want.abs() * 2.0 ** -24 + p * 2.0 ** -50).all())


@pytest.mark.parametrize("start", [0, 4000, 131000])
@pytest.mark.parametrize("rotary,hd,base", [(64, 64, 10000.0), (128, 128, 500000.0)])
def test_both_rotary_embeddings_agree_as_far_as_32_bits_of_an_angle_reach(start, rotary, hd, base):
    """A contiguous cache's tokens are turned by ``ops.rope``, whose frequencies and angles are of 32 bits: the exponent of the base, at most 13.2 in
    natural logarithms, and powf (4 steps), and their product leave an angle 13.2 + 8 + 1 half steps off, 23 * 2^-24 of itself; sines, products
    and sums add a few."""
    n, heads, hkv, page = 72, 2, 1, 16
    qkv = torch.randn(n, (heads + 2 * hkv) * hd, device="cuda")
    k, v = (torch.zeros(1, hkv, page, hd, device="cuda") for _ in range(2))
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    table = torch.zeros(1, (start + n) // page + 1, dtype=torch.int32, device="cuda")
    positions = [start + i if i < page else -1 for i in range(n)]            # (a page of them has a place)
    q, keys = ops.paged_append(qkv, k, v, table, ints(positions), heads, rows=ints([0] * n), rotary_dim=rotary, rope_base=base, keys=True)
    want = ops.rope(qkv[:page, :(heads + hkv) * hd].contiguous(), start, base, rotary, heads=heads + hkv).view(page, -1, hd)
    half = rotary // 2
    angle = (start + torch.arange(page, device="cuda").double())[:, None] * base ** (-2.0 * torch.arange(half, device="cuda").double() / rotary)
    x = qkv[:page, :(heads + hkv) * hd].view(page, -1, 2, half).double().abs().sum(2)
    bound = (x * (23 * angle + 8)[:, None] * 2.0 ** -24).repeat(1, 1, 2)
    assert bool(((torch.cat([q, keys], 1)[:page].double() - want.double()).abs() <= bound).all())
