"""The attention over the key/value cache (include/bnn_lowbit.h) where the
values of one head differ widely in size, on the GPU against its definition
in 64 bits.

Bounds, from the arithmetic alone, h = finfo(type).eps / 2, u = 2^-24:
- a score's error moves its weight by as much, relatively: twice that of all
  scores together, for the weight and for the sum;
- weight * scale is rounded to fp16 in a unit that puts the largest one that the
  row sees in the scale group at 2^8 at least: 2^-11 of it, or, below 2^-14,
  half of fp16's smallest step, 2^-25, which is 2^-33 of that largest one (times
  a code, at most `top`). Units end at 2^-118 of the largest weight: that is
  2^-143, as if no scale were below 2^-110;
- sums of n terms in 32 bits, in units that may cut: 2 n u of the terms'
  magnitudes, twice; 2^-20 for exponentials and joins;
- the result's own rounding: h, or half of its smallest subnormal number."""

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import bnns_to_c_b200 as bn  # noqa: E402

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
U = 2.0 ** -24


@pytest.fixture(scope="module", autouse=True)
def need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def whole(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def held(x, bits, group):
    """What a cache holds for x [n, heads, dim]: values and scales, exactly."""
    top, n = 2 ** (bits - 1) - 1, x.shape[-1]
    out, scales = torch.empty(x.shape, dtype=torch.float64, device="cuda"), []
    for at in range(0, n, group):
        part = x[..., at:at + group].double()
        s = (part.abs().amax(-1, keepdim=True) / top).to(torch.bfloat16).double()  # 8 bits: no tie of 64-bit quotients
        scales.append(s)
        out[..., at:at + group] = (part / s.clamp(min=1e-300)).round().clamp(-top, top) * s
    return out, torch.cat(scales, -1)


def check(q, k, v, bits, group, kind, cut, scale, page=16):
    """Attention of one sequence per row set of q [seqs, heads, dim] over the
    same keys and values; the first `cut` tokens as a shared prefix."""
    n, kv, dim = k.shape
    t, top, seqs = TYPES[kind], 2 ** (bits - 1) - 1, q.shape[0]
    pages = -(-n // page) + 2
    c = bn.KVCache(0, pages, page, kv, dim, bits=bits, group=group, dtype=kind)
    all_pages = torch.arange(pages, device="cuda", dtype=torch.int32)
    n_pre = -(-cut // page)
    pre, own = all_pages[:n_pre], all_pages[n_pre:][None].repeat(seqs, 1)
    if cut:
        c.write(k[:cut], v[:cut], pre[None], whole(0), offsets=whole(0, cut))
    c.write(k[cut:], v[cut:], own[:1], whole(0), offsets=whole(0, n - cut))
    out, lse = torch.full_like(q, 3.0), torch.full(q.shape[:2], 3.0, device="cuda")
    work = torch.full((c.attend_work(seqs, q.shape[1], cut),), 0xFF, device="cuda", dtype=torch.uint8)
    c.attend(q, torch.full((seqs,), n - cut, dtype=torch.int32, device="cuda"), own, out, work, lse=lse, scale=scale,
             prefix=pre if cut else None, prefix_tokens=cut)
    (kk, _), (vv, vs) = held(k, bits, group), held(v, bits, group)
    share = q.shape[1] // kv
    of = torch.arange(dim, device="cuda") // group
    for b in range(seqs):
        for h in range(q.shape[1]):
            x, keys, vals = q[b, h].double(), kk[:, h // share], vv[:, h // share]
            s = keys @ x * scale
            ds = (2 * (dim + 16) * U * (keys.abs() @ x.abs()) * abs(scale)).max() + 8 * U * s.abs().max()
            p = torch.softmax(s, 0)
            ref, size = p @ vals, p @ vals.abs()
            least = (p[:, None] * vs[:, h // share].clamp(min=2.0 ** -110)).amax(0)[of] * top * n * 2.0 ** -33
            tol = size * (2 * ds + 2 ** -11 + 2 ** -20 + 4 * n * U) + least
            f = torch.finfo(t)
            tol = tol + (f.eps / 2 * (ref.abs() + tol)).clamp(min=f.tiny * f.eps / 2)
            bad = ~((out[b, h].double() - ref).abs() <= tol)
            assert not bad.any(), (b, h, int(bad.sum()), int(bad.nonzero()[0]), out[b, h][bad][0].item(), ref[bad][0].item(), tol[bad][0].item())
            assert abs(lse[b, h].double() - torch.logsumexp(s, 0)) <= ds + 2 ** -20 + 2 * n * U + 4 * U * torch.logsumexp(s, 0).abs()


def aside(seed, n, kv, heads, dim, kind, at, score, ratio, own_rows=None):
    """Queries, keys and values of n tokens, of which token `at` has values
    `ratio` times the others' and a score `score` in every row (of own_rows;
    0 in the other rows). Channel 0 of the keys sets that score alone."""
    t = TYPES[kind]
    k, v = (torch.randn(n, kv, dim, device="cuda", generator=gen(seed + i)) for i in (1, 2))
    q = torch.randn(2, heads, dim, device="cuda", generator=gen(seed + 3)) * 0.3
    k[:, :, 0] = 0.0
    k[at] = 0.0
    k[at, :, 0] = 8.0
    q[:, :, 0] = score / 8.0
    if own_rows is not None:
        q[:, own_rows, 0] = 0.0
    v[at] *= ratio
    return q.to(t), k.to(t), v.to(t)


@pytest.mark.parametrize("at", [3, 200, 396])
@pytest.mark.parametrize("power", [10, 14, 17, 20, 24, 27, 30, 50])
def test_large_values_of_a_token_without_weight(power, at):
    """One token of 400 with values 2^power times the others' and a score 40
    (2^-58 of the weight) or 60 below theirs, in the first, a middle and the
    last block of 16."""
    score = -40.0 if power < 40 else -60.0
    for bits, group, dim in ((8, 64, 64), (4, 32, 128), (8, 32, 256)):
        q, k, v = aside(power, 400, 1, 4, dim, "bf16", at, score, 2.0 ** power)
        for cut in (0, 160):
            check(q, k, v, bits, group, "bf16", cut, 1.0)


@pytest.mark.parametrize("share", [1, 8, 16, 32])
def test_rows_of_a_tile_do_not_share_their_units(share):
    """The same, where half of a tile's rows do see the large values."""
    for bits, group, dim in ((8, 32, 128), (4, 64, 64), (4, 32, 192)):
        rows = torch.arange(0, share, 2)
        for at in (0, 130):
            q, k, v = aside(share, 200, 1, share, dim, "bf16", at, -40.0, 2.0 ** 26, own_rows=rows)
            check(q, k, v, bits, group, "bf16", 0, 1.0)
            check(q, k, v, bits, group, "bf16", 96, 1.0)


def test_large_values_first_in_the_range_of_fp16():
    """60000 beside 0.015, in fp16: the large ones first, with the highest
    score of the first blocks, and a later block that outweighs them by far."""
    n, dim = 256, 128
    k, v = (torch.randn(n, 2, dim, device="cuda", generator=gen(i)) for i in (1, 2))
    q = torch.randn(1, 16, dim, device="cuda", generator=gen(3)) * 0.1
    v = v.clamp(-3, 3) * 0.005
    v[:64] *= 4e6
    k[:, :, 0] = torch.arange(n, device="cuda")[:, None] // 64 * 1.0
    q[:, :, 0] = 40.0
    for bits, group in ((8, 128), (4, 32)):
        check(q.half(), k.half(), v.half(), bits, group, "fp16", 0, 1.0)
        check(q.half(), k.half(), v.half(), bits, group, "fp16", 80, 1.0)


def test_one_group_of_channels_far_larger():
    """Groups of one head differ by 2^40; each has a unit of its own."""
    n, dim = 300, 128
    k, v = (torch.randn(n, 1, dim, device="cuda", generator=gen(i)) for i in (5, 6))
    v[..., :32] *= 2.0 ** 30
    v[..., 64:96] *= 2.0 ** -10
    q = torch.randn(3, 8, dim, device="cuda", generator=gen(7)).to(torch.bfloat16)
    for bits in (8, 4):
        check(q, k.to(torch.bfloat16), v.to(torch.bfloat16), bits, 32, "bf16", 0, dim ** -0.5)


@pytest.mark.parametrize("power", [-132, -120, -60, 60, 110, 120])
def test_values_near_the_ends_of_bf16(power):
    """Sums of many values next to the largest and the smallest numbers: no
    product or sum on the way may leave the range of 32 bits."""
    for n in (40, 5000):
        k, v = (torch.rand(n, 1, 64, device="cuda", generator=gen(i)) + 0.5 for i in (1, 2))
        v = (v.double() * 2.0 ** power).to(torch.bfloat16)
        q = torch.randn(1, 8, 64, device="cuda", generator=gen(3)).to(torch.bfloat16)
        for cut in (0, 16):
            check(q, k.to(torch.bfloat16), v, 8, 64, "bf16", cut, 0.125)


def test_scores_that_rise_all_the_way():
    """Every block outweighs all before it, while the values shrink as fast,
    and the other way round."""
    n, dim = 480, 64
    for up in (True, False):
        k, v = (torch.randn(n, 1, dim, device="cuda", generator=gen(i)) for i in (1, 2))
        step = torch.arange(n, device="cuda") if up else torch.arange(n, device="cuda").flip(0)
        k[:, :, 0] = step[:, None] / 4.0  # exact in bf16 while below 64
        v = v * torch.exp2(-(step // 8).float())[:, None, None]
        q = torch.randn(1, 8, dim, device="cuda", generator=gen(3)) * 0.2
        q[:, :, 0] = torch.tensor([0.25, 0.5, 0.75, 1.0, 2.0, 0.0, -0.5, -2.0], device="cuda")
        for bits in (8, 4):
            check(q.to(torch.bfloat16), k.to(torch.bfloat16), v.to(torch.bfloat16), bits, 32, "bf16", 0, 1.0)
