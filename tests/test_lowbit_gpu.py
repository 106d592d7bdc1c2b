"""The low-bit operators (include/bnn_lowbit.h) on the GPU against their
definitions in 64 bits.

Tolerances, from the arithmetic alone. u = 2^-24 is half a step of 32 bits,
h = finfo(type).eps / 2 half a step of the result's type.
- A sum of n products in 32 bits, in any order, by units that may cut
  instead of round: at most 2 n u * sum |terms| off.
- A result rounded to its type: h * |result|, or half of the smallest
  subnormal number.
What else an operator rounds stands at its bound below."""

import math

import numpy as np
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


def rounding(ref, kind):
    """Half a step of `kind` at ref, and a little for ref's own neighbourhood."""
    f = torch.finfo(kind)
    return (f.eps / 2 * ref.abs()).clamp(min=f.tiny * f.eps / 2)


def within(got, ref, tol, what=""):
    got = got.double()
    off = (got - ref).abs() - tol
    bad = ~(off <= 0) & ~((got == ref) | (got.isnan() & ref.isnan()))
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()}, first at {bad.nonzero()[0].tolist()}, worst over by {off.nan_to_num().max().item():.3g}"


# ------------------------------------------------------------------ linear
def linear_case(seed, m, k, n, group, kind, zeros=False, bias=False):
    g, t = gen(seed), TYPES[kind]
    ng = -(-k // group)
    d = {"x": torch.randn(m, k, device="cuda", generator=g).to(t),
         "codes": torch.randint(0, 256, (n, (k + 1) // 2), device="cuda", generator=g, dtype=torch.uint8),
         "scales": (torch.rand(n, ng, device="cuda", generator=g) + 0.1).to(t),
         "zeros": torch.randint(0, 16, (n, ng), device="cuda", generator=g, dtype=torch.uint8) if zeros else None,
         "bias": torch.randn(n, device="cuda", generator=g) if bias else None}
    layer = bn.Q4Linear(0, k, n, d["codes"], d["scales"], zeros=d["zeros"], bias=d["bias"], group=group, dtype=kind)
    return layer, d


def linear_weights(d, k, group):
    c = d["codes"]
    q = torch.stack((c & 15, c >> 4), -1).flatten(1)[:, :k].double()
    of = torch.arange(k, device="cuda") // group
    z = d["zeros"].double()[:, of] if d["zeros"] is not None else 8.0
    return (q - z) * d["scales"].double()[:, of]


def linear_ref(d, x, k, group, kind):
    """Result and bound. Beside the sums: with more than 8 rows a weight
    (q - z) * s may be rounded to the type before it is multiplied, h * |x w|
    a term."""
    w = linear_weights(d, k, group)
    ref = x.double() @ w.T
    size = x.double().abs() @ w.abs().T
    if d["bias"] is not None:
        ref, size = ref + d["bias"].double(), size + d["bias"].double().abs()
    h = torch.finfo(TYPES[kind]).eps / 2 if x.shape[0] > 8 else 0.0
    tol = size * (2 * (k + 64) * U + h)
    return ref, tol + rounding(ref.abs() + tol, TYPES[kind])


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("m,k,n,group,zeros,bias", [
    (1, 1, 1, 32, False, False), (1, 31, 17, 32, True, False), (2, 33, 16, 32, True, True), (1, 64, 15, 64, False, True),
    (5, 96, 48, 96, True, False), (8, 200, 130, 64, False, False), (9, 130, 70, 128, True, True), (16, 512, 512, 128, False, False),
    (17, 1000, 77, 32, True, True), (33, 257, 129, 128, True, False), (64, 640, 300, 64, False, True), (65, 64, 64, 32, True, False),
    (100, 1030, 257, 128, True, True), (129, 448, 128, 64, True, True), (300, 777, 511, 32, True, True), (513, 256, 1000, 128, False, False),
    (1, 16384, 64, 128, True, False), (1, 120, 4096, 32, False, True),
    # long rows that TMA cannot load, at every width of a tile: many rounds of its stages
    (40, 4099, 200, 32, False, False), (60, 6002, 140, 128, True, False), (128, 5001, 130, 64, False, True), (260, 4098, 300, 128, True, True),
    (1000, 3001, 1111, 64, False, False),
    # K shared out in a cluster, at borders that are not a group's
    (1, 6464, 40, 256, True, False), (3, 4160, 16, 512, False, True), (12, 2176, 33, 128, True, True), (7, 8192, 100, 1024, True, False),
    # by three, five, six and seven, few rows and many, at every width of a tile
    (3, 4160, 100, 64, True, True), (5, 6464, 300, 32, False, False), (8, 9000, 90, 128, True, False), (1, 7168, 600, 256, True, True),
    (4, 5120, 2560, 512, False, True), (12, 3200, 100, 32, True, False), (10, 6464, 33, 128, True, True), (16, 9000, 300, 64, False, False),
    (70, 3200, 100, 32, True, True), (33, 2704, 90, 128, False, True), (200, 1800, 130, 64, True, False), (515, 2704, 130, 96, True, False),
    (65, 3264, 1000, 128, True, True), (1000, 1600, 300, 256, False, True), (700, 2704, 1000, 64, True, False)])
def test_linear(m, k, n, group, zeros, bias, kind):
    layer, d = linear_case(m * 7 + k, m, k, n, group, kind, zeros, bias)
    y = torch.full((m + 1, n), 7.0, device="cuda", dtype=TYPES[kind])
    layer.run(d["x"], y[:m])
    ref, tol = linear_ref(d, d["x"], k, group, kind)
    within(y[:m], ref, tol)
    assert (y[m] == 7).all()  # the row behind the last


@pytest.mark.parametrize("m", [1, 3, 40, 200])
def test_linear_strides_and_alignment(m):
    """Rows of x at an odd distance from an odd address, columns of a wider y."""
    k, n = 203, 90
    layer, d = linear_case(m, m, k, n, 64, "bf16", True, True)
    flat = torch.full((m * (k + 2) + 1,), float("nan"), device="cuda", dtype=torch.bfloat16)
    x = flat[1:].view(m, k + 2)[:, :k]
    x.copy_(d["x"])
    wide = torch.full((m, n + 7), -3.0, device="cuda", dtype=torch.bfloat16)
    layer.run(x, wide[:, 5:5 + n])
    ref, tol = linear_ref(d, d["x"], k, 64, "bf16")
    within(wide[:, 5:5 + n], ref, tol)
    assert (wide[:, :5] == -3).all() and (wide[:, 5 + n:] == -3).all()
    again = torch.empty(m, n, device="cuda", dtype=torch.bfloat16)
    layer.run(d["x"], again)  # the aligned path
    assert torch.equal(again, wide[:, 5:5 + n])


@pytest.mark.parametrize("m", [5, 18, 130])
def test_linear_padded_rows(m):
    """Rows of 200 of which 197 are x and the rest NaN, 16-byte aligned: what
    is behind a row's end is not read, or not used."""
    k, n = 197, 70
    layer, d = linear_case(m, m, k, n, 32, "fp16", True, False)
    x = torch.full((m, 200), float("nan"), device="cuda", dtype=torch.float16)
    x[:, :k] = d["x"]
    y = torch.empty(m, n, device="cuda", dtype=torch.float16)
    layer.run(x[:, :k], y)
    ref, tol = linear_ref(d, d["x"], k, 32, "fp16")
    within(y, ref, tol)


def test_linear_rows_far_apart():
    """The second row of x and of y 2^31 bytes and more behind the first."""
    k, n, far = 320, 64, (1 << 30) + 64
    layer, d = linear_case(1, 2, k, n, 64, "bf16", True, True)
    xs, ys = (torch.empty(far + 320, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    x, y = (t.as_strided((2, w), (far, 1)) for t, w in ((xs, k), (ys, n)))
    x.copy_(d["x"])
    layer.run(x, y)
    ref, tol = linear_ref(d, d["x"], k, 64, "bf16")
    within(y, ref, tol)


@pytest.mark.parametrize("m", [6, 150])
def test_linear_rows_do_not_mix(m):
    layer, d = linear_case(3, m, 320, 96, 64, "fp16", True, False)
    y0, y1 = (torch.empty(m, 96, device="cuda", dtype=torch.float16) for _ in range(2))
    layer.run(d["x"], y0)
    x = d["x"].clone()
    x[2, 17], x[4, 319] = float("nan"), float("inf")
    layer.run(x, y1)
    assert y1[2].isnan().all()
    w = linear_weights(d, 320, 64)[:, 319]
    assert torch.equal(y1[4].isnan(), w == 0) and torch.equal(y1[4].float().sign()[w != 0], w.float().sign()[w != 0])
    keep = [i for i in range(m) if i not in (2, 4)]
    assert torch.equal(y0[keep], y1[keep])


def test_linear_host_arrays_and_no_rows():
    layer, d = linear_case(8, 4, 100, 40, 32, "fp16", True, True)
    host = bn.Q4Linear(0, 100, 40, d["codes"].cpu().numpy(), d["scales"].cpu().numpy(), zeros=d["zeros"].cpu().numpy(),
                       bias=d["bias"].cpu(), group=32, dtype="fp16")
    y0, y1 = (torch.zeros(4, 40, device="cuda", dtype=torch.float16) for _ in range(2))
    layer.run(d["x"], y0)
    host.run(d["x"], y1)
    assert torch.equal(y0, y1)
    host.run(d["x"][:0], y1[:0])
    assert torch.equal(y0, y1)


@pytest.mark.parametrize("m", [2, 24, 400])
def test_linear_same_bits_every_time(m):
    layer, d = linear_case(m, m, 2048, 384, 128, "bf16", True, False)
    ys = [torch.empty(m, 384, device="cuda", dtype=torch.bfloat16) for _ in range(4)]
    for y in ys:
        layer.run(d["x"], y)
    assert all(torch.equal(ys[0], y) for y in ys)


# ------------------------------------------------------------------ cache
def quantise(x, bits, group):
    """The definition in 64 bits: codes and scales of x [.., dim]."""
    top, dim = 2 ** (bits - 1) - 1, x.shape[-1]
    codes, scales = torch.zeros(x.shape, dtype=torch.float64, device=x.device), []
    for at in range(0, dim, group):
        part = x[..., at:at + group].double()
        big = part.abs().amax(-1, keepdim=True)
        bad = ~torch.isfinite(part).all(-1, keepdim=True)
        # bf16 of the exact quotient, by integers: 8 bits of it, ties to even
        f, e = torch.frexp(torch.where(bad, 0.0, big) / top)
        least = -133  # the smallest bf16 step
        step = torch.maximum(e - 8, torch.full_like(e, least)).double()
        s = torch.exp2(step) * (f * torch.exp2(e.double() - step)).round()
        c = torch.where(s > 0, (part / torch.where(s > 0, s, 1.0)).round().clamp(-top, top), 0.0)
        codes[..., at:at + group] = torch.where(bad, 0.0, c)
        scales.append(torch.where(bad, float("nan"), s))
    return codes, torch.cat(scales, -1)


def values(codes, scales, group):
    return codes * scales.repeat_interleave(group, -1)[..., : codes.shape[-1]]


def ragged(lengths, start=None):
    off = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
    start = [0] * len(lengths) if start is None else start
    return torch.from_numpy(off).cuda(), torch.tensor(start, dtype=torch.int32, device="cuda")


def make_table(seed, seqs, width, pages):
    return torch.randperm(pages, device="cuda", generator=gen(seed))[: seqs * width].view(seqs, width).to(torch.int32)


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dim,group,page,heads", [(8, 0, 16, 1), (64, 32, 16, 2), (64, 0, 64, 1), (80, 32, 32, 3), (96, 0, 16, 2),
                                                  (128, 0, 64, 2), (128, 32, 128, 8), (136, 128, 16, 1), (192, 64, 256, 2),
                                                  (200, 32, 32, 1), (256, 0, 16, 2), (256, 128, 64, 1)])
def test_cache_write_and_read(dim, group, page, heads, bits, kind):
    """Ragged chunks at odd starts: every value is the definition's, bit for
    bit, and rows outside the sequences stay as they were."""
    lengths, start = [1, 0, 37, 16, 5], [3, 0, page - 1, 2 * page, 7]
    width = max(-(-(s + n) // page) for s, n in zip(start, lengths))
    c = bn.KVCache(0, 5 * width + 3, page, heads, dim, bits=bits, group=group, dtype=kind)
    table = make_table(dim, 5, width, 5 * width + 3)
    off, st = ragged(lengths, start)
    total = sum(lengths)
    x = [(torch.randn(total + 4, heads, dim, device="cuda", generator=gen(i)) * 3).to(TYPES[kind]) for i in (1, 2)]
    x[0][2, 0] *= 1000.0
    x[1][5] = 0.0
    c.write(*x, table, st, offsets=off)
    got = [torch.full_like(v, 5.0) for v in x]
    c.read(*got, table, st, offsets=off)
    for v, y in zip(x, got):
        ref = values(*quantise(v[:total], bits, group or dim), group or dim).to(TYPES[kind])
        assert torch.equal(y[:total], ref)
        assert (y[total:] == 5).all()


@pytest.mark.parametrize("bits", [8, 4])
def test_cache_extreme_values(bits):
    """Infinities and NaN spoil their own group alone; the smallest and the
    largest numbers of the type; ties."""
    big = torch.finfo(torch.bfloat16).max
    rows = torch.randn(10, 1, 96, device="cuda", generator=gen(5))
    rows[0, 0, 40], rows[1, 0, 3], rows[2, 0, 95] = float("inf"), float("nan"), -float("inf")
    rows[3], rows[4, 0, 1], rows[5] = 0.0, big, rows[5] * 1e-38
    rows[6] = rows[6] * 1e-40
    top = 2 ** (bits - 1) - 1
    rows[7] = (torch.arange(96, device="cuda") % (2 * top + 1) - top) * 0.5  # scale 0.5: every code, no rounding
    rows[8] = torch.where(torch.arange(96, device="cuda") % 2 == 0, 2.0 * top, 1.0)  # 1 / 2: a tie, to the even 0
    rows[9] = torch.where(torch.arange(96, device="cuda") % 2 == 0, 2.0 * top, -3.0)  # -3 / 2: to the even -2
    x = rows.to(torch.bfloat16)
    c = bn.KVCache(0, 1, 16, 1, 96, bits=bits, group=32, dtype="bf16")
    table, (off, st) = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), ragged([10])
    c.write(x, x, table, st, offsets=off)
    k, v = torch.empty_like(x), torch.empty_like(x)
    c.read(k, v, table, st, offsets=off)
    ref = values(*quantise(x, bits, 32), 32)
    ref = ref.to(torch.bfloat16)
    for y in (k, v):
        assert torch.equal(y.isnan(), ref.isnan()) and torch.equal(y.nan_to_num(), ref.nan_to_num())
    assert k[0, 0, 32:64].isnan().all() and not k[0, 0, :32].isnan().any() and k[2, 0, 64:].isnan().all()
    assert (k[8, 0, 1::2] == 0).all() and (k[9, 0, 1::2] == -4).all()


def test_cache_single_tokens_strides_and_overwriting():
    """One token a sequence without offsets, keys and values as views of one
    projection's output, twice over the same positions."""
    seqs, heads, dim = 9, 2, 64
    c = bn.KVCache(0, seqs, 16, heads, dim, bits=8, group=64, dtype="bf16")
    table = make_table(2, seqs, 1, seqs)
    start = torch.arange(seqs, device="cuda", dtype=torch.int32)
    for turn in range(2):
        qkv = torch.randn(seqs, 5 * heads * dim + 3, device="cuda", generator=gen(turn)).to(torch.bfloat16)
        k = qkv[:, 3:3 + heads * dim].unflatten(1, (heads, dim))
        v = qkv[:, 11 + heads * dim:11 + 3 * heads * dim].unflatten(1, (2 * heads, dim))[:, ::2]
        c.write(k, v, table, start)
    gk, gv = (torch.empty(heads, seqs, dim, device="cuda", dtype=torch.bfloat16).transpose(0, 1) for _ in range(2))
    c.read(gk, gv, table, start)
    for got, x in ((gk, k), (gv, v)):
        assert torch.equal(got, values(*quantise(x, 8, 64), 64).to(torch.bfloat16))
    # a position next to each written one is still what a new cache holds
    other = torch.full_like(gk, 9.0)
    c.read(other, gv, table, start + 1)
    assert (other == 0).all()


def test_cache_positions_without_a_page():
    """Entries outside the cache, positions before 0 and behind the table:
    not stored, not read, nothing else touched."""
    c = bn.KVCache(0, 3, 16, 1, 64, bits=8, dtype="fp16")
    x = torch.randn(64, 1, 64, device="cuda", generator=gen(1)).half()
    whole = torch.tensor([[0, 1, 2]], dtype=torch.int32, device="cuda")
    off, st = ragged([48])
    c.write(x[:48], x[:48], whole, st, offsets=off)
    k0, v0 = torch.empty_like(x[:48]), torch.empty_like(x[:48])
    c.read(k0, v0, whole, st, offsets=off)
    for table in ([[-1, 3, 1 << 30]], [[-2 ** 31, 2 ** 31 - 1, -7]]):
        table = torch.tensor(table, dtype=torch.int32, device="cuda")
        for start in (0, -70, 2 ** 31 - 10, -2 ** 31, 48, 40):
            off, st = ragged([64], [start])
            c.write(x * 2, x * 2, table, st, offsets=off)
            y = torch.full_like(x, 3.0)
            c.read(y, y.clone(), table, st, offsets=off)
            assert (y == 3).all()
    off, st = ragged([30], [40])  # 8 inside, 22 behind the table
    y = torch.full((30, 1, 64), 3.0, device="cuda", dtype=torch.float16)
    c.read(y, y.clone(), whole, st, offsets=off)
    assert torch.equal(y[:8], k0[40:]) and (y[8:] == 3).all()
    k1, v1 = torch.empty_like(k0), torch.empty_like(v0)
    off, st = ragged([48])
    c.read(k1, v1, whole, st, offsets=off)
    assert torch.equal(k0, k1) and torch.equal(v0, v1)


# ------------------------------------------------------------------ attention
def filled(seed, lengths, heads, dim, bits, group, kind, page, prefix=0, spare=2, mag=1.0):
    """A cache with sequences of these lengths (and a prefix), and what it
    holds in 64 bits: a list of [length, heads, dim] keys and values."""
    t, g = TYPES[kind], group or dim
    width = max(1, -(-max(lengths + [1]) // page))
    n_pre = -(-prefix // page)
    pages = len(lengths) * width + n_pre + spare
    c = bn.KVCache(0, pages, page, heads, dim, bits=bits, group=group, dtype=kind)
    order = torch.randperm(pages, device="cuda", generator=gen(seed)).to(torch.int32)
    table = order[: len(lengths) * width].view(len(lengths), width).contiguous()
    pre = order[len(lengths) * width:][:n_pre].contiguous()
    # what earlier users left in the pages, NaN among it, is not to be seen
    junk = torch.full((pages * page, heads, dim), float("nan"), device="cuda", dtype=t)
    off, st = ragged([pages * page])
    c.write(junk, junk, order[None], st, offsets=off)
    total = sum(lengths) + prefix
    x = [(torch.randn(total, heads, dim, device="cuda", generator=gen(seed + i)) * mag).to(t) for i in (1, 2)]
    off, st = ragged(lengths)
    if sum(lengths):
        c.write(x[0][prefix:], x[1][prefix:], table, st, offsets=off)
    if prefix:
        off, st = ragged([prefix])
        c.write(x[0][:prefix], x[1][:prefix], pre[None], st, offsets=off)
    kv = [values(*quantise(v, bits, g), g) for v in x]
    at, held = prefix, []
    for n in lengths:
        held.append(tuple(torch.cat((v[:prefix], v[at:at + n])) for v in kv))
        at += n
    return c, table, pre, held


def attend_ref(q, held, scale, kind):
    """Results, log-sums and bounds. exp(s) has the relative error of s's
    absolute one; weights are rounded to fp16 (2^-12, or 2^-25 of a unit that
    is at most twice the largest scale: |value| <= 127 scales, so at most
    2^-23 of the largest |value| a token); 2^-21 for exp2 and the joins."""
    b, heads, dim = q.shape
    out = torch.zeros(b, heads, dim, dtype=torch.float64, device="cuda")
    lse = torch.full((b, heads), -math.inf, dtype=torch.float64, device="cuda")
    t_out, t_lse = torch.zeros_like(out), torch.zeros_like(lse)
    for i, (k, v) in enumerate(held):
        if not k.shape[0]:
            continue
        share = heads // k.shape[1]
        for h in range(heads):
            kk, vv = k[:, h // share], v[:, h // share]
            x = q[i, h].double()
            s = kk @ x * scale
            size = kk.abs() @ x.abs() * abs(scale)
            ds = (2 * (dim + 16) * U * size).max() + 8 * U * s.abs().max()
            p = torch.softmax(s, 0)
            n = k.shape[0]
            d = 2 * ds + 2 ** -12 + 2 ** -21 + 4 * n * U
            lse[i, h], t_lse[i, h] = torch.logsumexp(s, 0), ds + 2 ** -21 + 2 * n * U + 4 * U * torch.logsumexp(s, 0).abs()
            out[i, h], t_out[i, h] = p @ vv, d * (p @ vv.abs()) + n * 2.0 ** -23 * vv.abs().max()
    return out, lse, t_out + rounding(out.abs() + t_out, TYPES[kind]), t_lse


def attend(c, q, lengths, table, prefix=None, prefix_tokens=0, scale=None, poison=0xFF, stream=None):
    out = torch.full_like(q, 3.0)
    lse = torch.full(q.shape[:2], 3.0, device="cuda")
    work = torch.full((c.attend_work(q.shape[0], q.shape[1], prefix_tokens),), poison, device="cuda", dtype=torch.uint8)
    c.attend(q, torch.tensor(lengths, dtype=torch.int32, device="cuda"), table, out, work, lse=lse, scale=scale,
             prefix=prefix, prefix_tokens=prefix_tokens, stream=stream)
    return out, lse


def check_attend(seed, lengths, heads, share, dim, bits, group, kind, page, prefix=0, mag=1.0, scale=None):
    c, table, pre, held = filled(seed, lengths, heads, dim, bits, group, kind, page, prefix, mag=mag)
    q = torch.randn(len(lengths), heads * share, dim, device="cuda", generator=gen(seed + 9)).to(TYPES[kind])
    out, lse = attend(c, q, lengths, table, pre if prefix else None, prefix, scale)
    r_out, r_lse, t_out, t_lse = attend_ref(q, held, dim ** -0.5 if scale is None else scale, kind)
    within(out, r_out, t_out, "out")
    within(lse, r_lse, t_lse, "lse")


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dim,group,share,heads,page", [
    (64, 0, 1, 1, 16), (64, 32, 4, 2, 64), (128, 0, 8, 2, 64), (128, 32, 6, 1, 32), (128, 64, 16, 2, 128), (80, 32, 3, 3, 16),
    (96, 0, 20, 1, 64), (8, 0, 2, 1, 16), (136, 128, 8, 1, 32), (192, 64, 12, 2, 16), (256, 0, 5, 1, 256), (256, 32, 33, 1, 64)])
def test_attend_head_layouts(dim, group, share, heads, page, bits, kind):
    check_attend(dim + share, [130, 1, 0, 77], heads, share, dim, bits, group, kind, page)


@pytest.mark.parametrize("length", [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 255, 257, 1000, 4097])
def test_attend_lengths(length):
    check_attend(length, [length], 2, 4, 128, 8, 0, "bf16", 32)
    check_attend(length + 1, [length, 3, length], 1, 8, 64, 4, 32, "fp16", 16)


def test_attend_all_empty():
    check_attend(3, [0, 0, 0, 0, 0], 2, 4, 64, 8, 0, "fp16", 16)


def test_attend_ragged_batch():
    rng = np.random.default_rng(4)
    lengths = [int(n) for n in rng.integers(0, 900, 40)] + [6000]
    check_attend(11, lengths, 2, 8, 128, 4, 32, "bf16", 64)


@pytest.mark.parametrize("heads", [1, 8])
def test_attend_long(heads):
    check_attend(5, [20011], heads, 8, 128, 8, 128, "bf16", 64)


@pytest.mark.parametrize("prefix,lengths,heads,share,dim,bits,kind", [
    (1, [0, 0], 1, 1, 64, 8, "fp16"), (16, [0, 1, 2], 2, 4, 64, 4, "bf16"), (100, [5, 0, 70], 2, 8, 128, 8, "bf16"),
    (257, [0] * 7, 1, 3, 80, 8, "fp16"), (3000, [31, 900, 0, 1], 4, 4, 128, 4, "fp16"), (600, list(range(40)), 2, 4, 64, 8, "fp16"),
    (513, [9] * 20, 1, 2, 256, 8, "bf16"), (40, [3] * 3, 1, 50, 192, 4, "bf16")])
def test_attend_shared_prefix(prefix, lengths, heads, share, dim, bits, kind):
    check_attend(prefix, lengths, heads, share, dim, bits, 32, kind, 16, prefix=prefix)


@pytest.mark.parametrize("prefix,length", [(0, 700), (90, 5), (300, 0), (1030, 300)])
@pytest.mark.parametrize("seqs,dim,kind", [(100, 64, "bf16"), (480, 80, "fp16"), (130, 256, "bf16")])
def test_attend_many_rows(seqs, dim, kind, prefix, length):
    """Thousands of query rows, all of one sequence (and of an empty one), so
    that one reference serves; rows of the output at an odd distance."""
    heads, share = 2, 8
    c, table, pre, held = filled(seqs, [length], heads, dim, 4, 32, kind, 16, prefix)
    q1 = torch.randn(1, heads * share, dim, device="cuda", generator=gen(4)).to(TYPES[kind])
    r_out, r_lse, t_out, t_lse = attend_ref(q1, held, dim ** -0.5, kind)
    lengths = torch.full((seqs,), length, dtype=torch.int32, device="cuda")
    lengths[7] = 0
    work = torch.full((c.attend_work(seqs, heads * share, prefix),), 0xFF, device="cuda", dtype=torch.uint8)
    wide = torch.full((seqs, heads * share, dim + 3), 3.0, device="cuda", dtype=TYPES[kind])
    out, lse = wide[:, :, 1:dim + 1], torch.full((seqs, heads * share), 3.0, device="cuda")
    c.attend(q1.expand(seqs, -1, -1), lengths, table.expand(seqs, -1).contiguous(), out, work, lse=lse,
             prefix=pre if prefix else None, prefix_tokens=prefix)
    assert (wide[:, :, 0] == 3).all() and (wide[:, :, dim + 1:] == 3).all()
    others = [i for i in range(seqs) if i != 7]
    within(out[others], r_out.expand(seqs - 1, -1, -1), t_out.expand(seqs - 1, -1, -1), "out")
    within(lse[others], r_lse.expand(seqs - 1, -1), t_lse.expand(seqs - 1, -1), "lse")
    r_out, r_lse, t_out, t_lse = attend_ref(q1, [tuple(x[:prefix] for x in held[0])], dim ** -0.5, kind)
    within(out[7:8], r_out, t_out, "out of the empty one")
    within(lse[7:8], r_lse, t_lse, "lse of the empty one")


@pytest.mark.parametrize("mag", [1e-3, 40.0, 1e4])
def test_attend_magnitudes(mag):
    """Flat and peaked weights; values far from one in size."""
    check_attend(7, [500, 90], 2, 4, 64, 8, 0, "bf16", 16, mag=mag, scale=0.3 / mag)
    check_attend(8, [500, 90], 2, 4, 64, 4, 32, "bf16", 16, mag=mag, scale=0.02)


def test_attend_scales_of_values_grow_and_fall():
    """Later values 2^12 times the earlier, and the other way round: the unit
    that sums are kept in has to follow."""
    for flip in (False, True):
        n, dim = 400, 64
        c = bn.KVCache(0, 25, 16, 1, dim, bits=8, group=32, dtype="bf16")
        k = torch.randn(n, 1, dim, device="cuda", generator=gen(1)).to(torch.bfloat16)
        size = torch.exp2(torch.linspace(-6, 6, n, device="cuda")).flip(0) if flip else torch.exp2(torch.linspace(-6, 6, n, device="cuda"))
        v = (torch.randn(n, 1, dim, device="cuda", generator=gen(2)) * size[:, None, None]).to(torch.bfloat16)
        table = torch.arange(25, device="cuda", dtype=torch.int32)[None]
        off, st = ragged([n])
        c.write(k, v, table, st, offsets=off)
        q = torch.randn(1, 4, dim, device="cuda", generator=gen(3)).to(torch.bfloat16)
        out, lse = attend(c, q, [n], table)
        held = [tuple(values(*quantise(x, 8, 32), 32) for x in (k, v))]
        r_out, r_lse, t_out, t_lse = attend_ref(q, held, dim ** -0.5, "bf16")
        within(out, r_out, t_out)
        within(lse, r_lse, t_lse)


def test_attend_nan_in_view_and_out_of_it():
    """A NaN key or value that is seen makes its rows NaN; one behind the
    length (or of another kv head) does not."""
    lengths = [100, 100]
    c, table, _, held = filled(3, lengths, 2, 64, 8, 0, "fp16", 16)
    q = torch.randn(2, 8, 64, device="cuda", generator=gen(1)).half()
    base, _ = attend(c, q, lengths, table)
    assert not base.isnan().any()  # pages behind the lengths hold NaN already
    one = torch.zeros(1, 2, 64, device="cuda", dtype=torch.float16)
    one[0, 1, 5] = float("nan")  # head 1
    at = torch.tensor([50], dtype=torch.int32, device="cuda")
    k, v = (torch.empty(1, 2, 64, device="cuda", dtype=torch.float16) for _ in range(2))
    c.read(k, v, table[1:2], at)
    c.write(k + one, v, table[1:2], at)
    out, lse = attend(c, q, lengths, table)
    assert out[1, 4:].isnan().all() and lse[1, 4:].isnan().all()
    assert torch.equal(out[0], base[0]) and not out[1, :4].isnan().any()
    c.write(k, v + one, table[1:2], at)
    out, lse = attend(c, q, lengths, table)
    assert out[1, 4:].isnan().all() and not lse.isnan().any() and torch.equal(out[0], base[0])
    out, _ = attend(c, q, [100, 50], table)
    assert not out.isnan().any()


def test_attend_only_nan_is_not_empty():
    c = bn.KVCache(0, 1, 16, 1, 64, bits=8, dtype="bf16")
    x = torch.full((1, 1, 64), float("nan"), device="cuda", dtype=torch.bfloat16)
    table, at = (torch.zeros(*s, dtype=torch.int32, device="cuda") for s in ((1, 1), (1,)))
    c.write(x, x, table, at)
    out, lse = attend(c, torch.ones(1, 1, 64, device="cuda", dtype=torch.bfloat16), [1], table)
    assert out.isnan().all() and lse.isnan().all()


@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
@pytest.mark.parametrize("prefix", [0, 40])
def test_attend_query_that_is_not_finite(bad, prefix):
    """Its scores are infinities of one sign at best: the softmax is NaN, in
    that row alone; one that sees nothing is still empty."""
    c = bn.KVCache(0, 8, 16, 1, 64, bits=8, dtype="bf16")
    x = torch.rand(80, 1, 64, device="cuda", generator=gen(1)).to(torch.bfloat16) + 0.5
    own, pre = (torch.arange(a, b, dtype=torch.int32, device="cuda") for a, b in ((0, 5), (5, 8)))
    for pages, n in ((own, 80), (pre, 40)):
        c.write(x[:n], x[:n], pages[None], torch.zeros(1, dtype=torch.int32, device="cuda"),
                offsets=torch.tensor([0, n], dtype=torch.int32, device="cuda"))
    q = torch.randn(2, 4, 64, device="cuda", generator=gen(2)).to(torch.bfloat16)
    table, args = own[None].repeat(2, 1), (pre, prefix) if prefix else ()
    base, base_lse = attend(c, q, [80, 0], table, *args)
    q[:, 2, 7] = bad
    out, lse = attend(c, q, [80, 0], table, *args)
    for b in range(2):
        for i in range(4):
            if i == 2 and (b == 0 or prefix):
                assert out[b, i].isnan().all() and lse[b, i].isnan()
            else:
                assert torch.equal(out[b, i], base[b, i]) and lse[b, i] == base_lse[b, i]
    if not prefix:
        assert (out[1] == 0).all() and (lse[1] == -math.inf).all()


def test_attend_missing_pages_and_odd_lengths():
    """Positions without a page are not there: in the middle, at the end,
    behind the table, in the prefix; a negative length is an empty one."""
    page = 16
    c, table, pre, held = filled(21, [100, 64, 40], 1, 64, 8, 0, "bf16", page, prefix=48)
    q = torch.randn(3, 4, 64, device="cuda", generator=gen(2)).to(torch.bfloat16)
    t2, p2 = table.clone(), pre.clone()
    t2[0, 2], t2[0, 6], t2[1] = -1, 10 ** 9, torch.tensor([-5, 2 ** 31 - 1, -2 ** 31, 99, -1, -1, -1], device="cuda")
    p2[1] = -1
    out, lse = attend(c, q, [100, 64, 40], t2, p2, 48)
    keep0 = [i for i in range(148) if not (16 <= i < 32) and not (48 + 32 <= i < 48 + 48) and i < 48 + 96]
    keep1 = [i for i in range(48) if not 16 <= i < 32]
    keep2 = [i for i in range(88) if not 16 <= i < 32]
    kept = [tuple(x[k] for x in h) for h, k in zip(held, (keep0, keep1, keep2))]
    r_out, r_lse, t_out, t_lse = attend_ref(q, kept, 0.125, "bf16")
    within(out, r_out, t_out)
    within(lse, r_lse, t_lse)
    # lengths beyond the table count up to its end; the last pages hold NaN behind position 100 of sequence 0
    out, lse = attend(c, q[1:], [-3, -2 ** 31], table[1:])
    assert (out == 0).all() and (lse == -math.inf).all()
    full, lse = attend(c, q[:1], [2 ** 31 - 1], table[:1])
    assert full.isnan().all()
    none = torch.zeros(3, 0, dtype=torch.int32, device="cuda")
    out, lse = attend(c, q, [5, 5, 5], none)
    assert (out == 0).all() and (lse == -math.inf).all()


def test_attend_strides_and_neighbours():
    lengths, heads, share, dim = [70, 20], 2, 3, 80
    c, table, _, held = filled(31, lengths, heads, dim, 8, 32, "fp16", 16)
    qkv = torch.randn(2, 10 * dim + 1, device="cuda", generator=gen(4)).half()
    q = qkv[:, 1:1 + 6 * dim].unflatten(1, (6, dim))
    buf = torch.full((2, 6, dim + 9), 4.0, device="cuda", dtype=torch.float16)
    out = buf[:, :, 3:3 + dim]
    work = torch.empty(c.attend_work(2, 6), device="cuda", dtype=torch.uint8)
    c.attend(q, torch.tensor(lengths, dtype=torch.int32, device="cuda"), table, out, work)
    r_out, _, t_out, _ = attend_ref(q, held, dim ** -0.5, "fp16")
    within(out, r_out, t_out)
    assert (buf[:, :, :3] == 4).all() and (buf[:, :, 3 + dim:] == 4).all()


def test_attend_whatever_the_workspace_holds():
    c, table, pre, _ = filled(41, [300, 0, 2000], 2, 64, 8, 0, "bf16", 16, prefix=90)
    q = torch.randn(3, 8, 64, device="cuda", generator=gen(5)).to(torch.bfloat16)
    for prefix in (0, 90):
        got = [attend(c, q, [300, 0, 2000], table, pre if prefix else None, prefix, poison=b) for b in (0, 0xFF, 0x7F)]
        for out, lse in got[1:]:
            assert torch.equal(out, got[0][0]) and torch.equal(lse, got[0][1])


# ------------------------------------------------------------------ streams, graphs, a decode step
def step_state(seed, seqs=4, heads=2, share=4, dim=64, hidden=192):
    """The weights and the cache of one layer's decode step."""
    kind = torch.bfloat16
    mk = lambda s, k, n: linear_case(s, 1, k, n, 64, "bf16", True, True)  # noqa: E731
    (qkv, dq), (proj, dp) = mk(seed, hidden, (heads * share + 2 * heads) * dim), mk(seed + 1, heads * share * dim, hidden)
    c, table, _, _ = filled(seed, [40, 7, 0, 63], heads, dim, 8, 0, "bf16", 16)
    width = table.shape[1] + 2
    grown = torch.full((seqs, width), -1, dtype=torch.int32, device="cuda")
    grown[:, : table.shape[1]] = table
    return {"qkv": qkv, "proj": proj, "dq": dq, "dp": dp, "cache": c, "table": grown, "hidden": hidden, "heads": heads, "share": share,
            "dim": dim, "x": torch.randn(seqs, hidden, device="cuda", generator=gen(seed + 2)).to(kind),
            "lengths": torch.tensor([40, 7, 0, 62], dtype=torch.int32, device="cuda"),
            "y": torch.empty(seqs, (heads * share + 2 * heads) * dim, device="cuda", dtype=kind),
            "a": torch.empty(seqs, heads * share, dim, device="cuda", dtype=kind), "o": torch.empty(seqs, hidden, device="cuda", dtype=kind),
            "work": torch.empty(c.attend_work(seqs, heads * share), device="cuda", dtype=torch.uint8), "len1": torch.empty(seqs, dtype=torch.int32, device="cuda")}


def step(s, stream=None):
    """Projection, store, attention, projection: one decode step."""
    h, d, g = s["heads"], s["dim"], s["share"]
    s["qkv"].run(s["x"], s["y"], stream=stream)
    q, k, v = s["y"].unflatten(1, (-1, d)).split((h * g, h, h), 1)
    s["cache"].write(k, v, s["table"], s["lengths"], stream=stream)
    s["len1"].copy_(s["lengths"] + 1)
    s["cache"].attend(q, s["len1"], s["table"], s["a"], s["work"], stream=stream)
    s["proj"].run(s["a"].flatten(1), s["o"], stream=stream)


def step_ref(s, before):
    """The step from its own intermediate results, each in 64 bits."""
    h, d, g, kind = s["heads"], s["dim"], s["share"], torch.bfloat16
    ref, tol = linear_ref(s["dq"], s["x"], s["hidden"], 64, "bf16")
    within(s["y"], ref, tol, "qkv")
    q, k, v = s["y"].unflatten(1, (-1, d)).split((h * g, h, h), 1)
    held = []
    for b, n in enumerate(s["lengths"].tolist()):
        held.append(tuple(torch.cat((old[b][:n], values(*quantise(x[b:b + 1], 8, d), d))) for old, x in zip(before, (k, v))))
    r_out, _, t_out, _ = attend_ref(q, held, d ** -0.5, "bf16")
    within(s["a"], r_out, t_out, "attention")
    ref, tol = linear_ref(s["dp"], s["a"].flatten(1).to(kind), h * g * d, 64, "bf16")
    within(s["o"], ref, tol, "projection")


def test_decode_step_eager_and_captured():
    """A run of the operators together, eagerly on a side stream and as a
    captured graph that is replayed on new inputs."""
    s = step_state(50)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(s, stream=side)
    torch.cuda.synchronize()
    eager = [s[k].clone() for k in ("y", "a", "o")]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        step(s, stream=torch.cuda.current_stream())
    for k in ("y", "a", "o"):
        s[k].zero_()
    g.replay()
    torch.cuda.synchronize()
    for a, k in zip(eager, ("y", "a", "o")):
        assert torch.equal(a, s[k])
    s["x"].copy_(torch.randn_like(s["x"].float()).to(torch.bfloat16))
    s["lengths"].copy_(torch.tensor([39, 8, 1, 60], dtype=torch.int32))
    g.replay()
    torch.cuda.synchronize()
    replayed = [s[k].clone() for k in ("y", "a", "o")]
    step(s)
    torch.cuda.synchronize()
    for a, k in zip(replayed, ("y", "a", "o")):
        assert torch.equal(a, s[k])


def test_decode_step_against_the_definitions():
    s = step_state(60)
    # what the cache holds, exactly: written again from values that 8 bits hold without loss
    seqs, n = s["table"].shape[0], 64
    x = [(torch.randint(-127, 128, (seqs * n, s["heads"], s["dim"]), device="cuda", generator=gen(i)) / 64).to(torch.bfloat16) for i in (1, 2)]
    for v in x:
        v[..., 0] = 127 / 64  # scale 1 / 64 in every head
    at = torch.arange(seqs + 1, device="cuda", dtype=torch.int32) * n
    s["cache"].write(*x, s["table"], torch.zeros(seqs, dtype=torch.int32, device="cuda"), offsets=at)
    before = [v.double().view(seqs, n, s["heads"], s["dim"]) for v in x]
    step(s)
    torch.cuda.synchronize()
    step_ref(s, before)


def test_steps_in_a_row_as_each_alone():
    """Sixty steps without a wait between them, each reading what the one
    before it has written, against the same steps with a wait after each
    kernel: the kernels' early starts overlap nothing that they must not."""
    s, t = step_state(80), step_state(80)
    xs = [torch.randn(4, s["hidden"], device="cuda", generator=gen(90 + i)).to(torch.bfloat16) for i in range(60)]
    outs = []
    for v, waits in ((s, False), (t, True)):
        got = [torch.empty_like(v["o"]) for _ in xs]
        torch.cuda.synchronize()
        for i, x in enumerate(xs):
            v["x"].copy_(x)
            v["lengths"].fill_(i % 50)
            v["qkv"].run(v["x"], v["y"])
            if waits:
                torch.cuda.synchronize()
            q, k, w = v["y"].unflatten(1, (-1, 64)).split((8, 2, 2), 1)
            v["cache"].write(k, w, v["table"], v["lengths"])
            if waits:
                torch.cuda.synchronize()
            v["len1"].copy_(v["lengths"] + 1)
            v["cache"].attend(q, v["len1"], v["table"], v["a"], v["work"])
            if waits:
                torch.cuda.synchronize()
            v["proj"].run(v["a"].flatten(1), v["o"])
            v["proj"].run(v["a"].flatten(1), got[i])
            v["x"].add_(v["o"])  # the next projection's input, from this one's output
            v["qkv"].run(v["x"], v["y"])
            if waits:
                torch.cuda.synchronize()
            got[i].add_(v["y"][:, :192])
        torch.cuda.synchronize()
        outs.append(got)
    assert all(torch.equal(a, b) for a, b in zip(*outs))


def test_captured_attention_behind_a_prefix():
    """Two graphs of one cache, each with a workspace of its own, replayed on
    two streams at once on new queries."""
    lengths = [70, 0, 400]
    c, table, pre, held = filled(91, lengths, 2, 64, 8, 0, "fp16", 16, prefix=200)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    sides = []
    for i in range(2):
        q = torch.randn(3, 8, 64, device="cuda", generator=gen(i)).half()
        out, work = torch.empty_like(q), torch.empty(c.attend_work(3, 8, 200), device="cuda", dtype=torch.uint8)
        st = torch.cuda.Stream()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            c.attend(q, n, table, out, work, prefix=pre, prefix_tokens=200, stream=torch.cuda.current_stream())
        sides.append((g, q, out, work, st))
    for turn in range(3):
        for i, (g, q, out, work, st) in enumerate(sides):
            q.copy_(torch.randn(3, 8, 64, device="cuda", generator=gen(10 * turn + i)).half())
        torch.cuda.synchronize()
        for g, q, out, work, st in sides:
            with torch.cuda.stream(st):
                for _ in range(5):
                    g.replay()
        torch.cuda.synchronize()
        for g, q, out, work, st in sides:
            r_out, _, t_out, _ = attend_ref(q, held, 0.125, "fp16")
            within(out, r_out, t_out)


def test_cache_beyond_four_gigabytes():
    """Pages whose codes lie 2^32 bytes and more from the first."""
    c = bn.KVCache(0, 34000, 64, 8, 256, bits=8, group=128, dtype="bf16")
    assert c.nbytes > 2 * 2 ** 32
    table = torch.tensor([[33999, 3, 33001], [33500, 20000, 1]], dtype=torch.int32, device="cuda")
    lengths = [150, 131]
    off, st = ragged(lengths)
    x = [torch.randn(281, 8, 256, device="cuda", generator=gen(i)).to(torch.bfloat16) for i in (1, 2)]
    c.write(*x, table, st, offsets=off)
    got = [torch.empty_like(v) for v in x]
    c.read(*got, table, st, offsets=off)
    kv = [values(*quantise(v, 8, 128), 128) for v in x]
    for v, y in zip(kv, got):
        assert torch.equal(y, v.to(torch.bfloat16))
    q = torch.randn(2, 8, 256, device="cuda", generator=gen(3)).to(torch.bfloat16)
    out, lse = attend(c, q, lengths, table)
    held = [tuple(v[a:b] for v in kv) for a, b in ((0, 150), (150, 281))]
    r_out, r_lse, t_out, t_lse = attend_ref(q, held, 256 ** -0.5, "bf16")
    within(out, r_out, t_out)
    within(lse, r_lse, t_lse)


def test_two_streams_at_once():
    """Two caches' worth of attention on two streams, each with a workspace
    of its own, and one layer used from both."""
    c, table, _, _ = filled(71, [700, 1200], 2, 64, 8, 0, "bf16", 16)
    layer, d = linear_case(5, 8, 512, 256, 64, "bf16", True, True)
    q = [torch.randn(2, 8, 64, device="cuda", generator=gen(i)).to(torch.bfloat16) for i in (1, 2)]
    want = [attend(c, x, [700, 1200], table) for x in q]
    xs = [d["x"], d["x"].flip(0).contiguous()]
    wy = [torch.empty(8, 256, device="cuda", dtype=torch.bfloat16) for _ in xs]
    for x, y in zip(xs, wy):
        layer.run(x, y)
    lengths = torch.tensor([700, 1200], dtype=torch.int32, device="cuda")
    outs = [[torch.empty_like(x) for _ in range(10)] for x in q]
    ys = [[torch.empty_like(y) for _ in range(10)] for y in wy]
    works = [torch.empty(c.attend_work(2, 8), device="cuda", dtype=torch.uint8) for _ in q]
    streams = [torch.cuda.Stream() for _ in q]
    torch.cuda.synchronize()
    for i in range(10):
        for k, st in enumerate(streams):
            c.attend(q[k], lengths, table, outs[k][i], works[k], stream=st)
            layer.run(xs[k], ys[k][i], stream=st)
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(o, want[k][0]) for o in outs[k])
        assert all(torch.equal(y, wy[k]) for y in ys[k])


def test_failing_allocations_are_reported():
    free = torch.cuda.mem_get_info()[0]
    codes, scales = np.zeros((16, 32), np.uint8), np.zeros((16, 2), np.uint16)
    try:
        for k in (1, 2):
            bn.inject_fault(bn.FAULT_ALLOC, k)
            with pytest.raises(bn.BnnError) as e:
                bn.Q4Linear(0, 64, 16, codes, scales, group=32)
            assert e.value.code == bn.BNN_ERR_OOM
        bn.inject_fault(bn.FAULT_ALLOC, 1)
        with pytest.raises(bn.BnnError) as e:
            bn.KVCache(0, 64, 16, 1, 64)
        assert e.value.code == bn.BNN_ERR_OOM
    finally:
        bn.inject_fault(0)
    assert torch.cuda.mem_get_info()[0] == free


# ------------------------------------------------------------------ weights outside the type's range
@pytest.mark.parametrize("kind,scale", [("fp16", 8000.0), ("bf16", 2.0 ** 125)])
@pytest.mark.parametrize("m", [1, 9, 16, 17, 40, 300, 1000])
def test_linear_weights_beyond_the_type(m, kind, scale):
    """(q - z) * s leaves the type's range for some weights of a layer; the
    results do not, with any number of rows. Such a layer's weights are never
    rounded: a group's scale is applied to its 32-bit sum."""
    k, n, group = 640, 136, 64
    _, d = linear_case(m, m, k, n, group, kind, True, True)
    d["scales"][5::16] = (d["scales"][5::16].float() * scale).to(TYPES[kind])
    layer = bn.Q4Linear(0, k, n, d["codes"], d["scales"], zeros=d["zeros"], bias=d["bias"], group=group, dtype=kind)
    x = (d["x"].float() * 2.0 ** -10).to(TYPES[kind])
    y = torch.full((m + 1, n), 7.0, device="cuda", dtype=TYPES[kind])
    layer.run(x, y[:m])
    w = linear_weights(d, k, group)
    assert (w.abs() > torch.finfo(TYPES[kind]).max).any()
    ref, size = x.double() @ w.T + d["bias"].double(), x.double().abs() @ w.abs().T + d["bias"].double().abs()
    assert ref.abs().max() < torch.finfo(TYPES[kind]).max
    tol = size * (2 * (k + 64) * U)
    within(y[:m], ref, tol + rounding(ref.abs() + tol, TYPES[kind]))
    assert (y[m] == 7).all()


@pytest.mark.parametrize("scale,zero", [(65504 / 15 - 2, 0), (4370.0, 0), (65504 / 7 - 4, 8), (9368.0, 8)])
def test_linear_weights_next_to_the_end_of_the_type(scale, zero):
    """The largest weight just inside and just outside of fp16."""
    scales = torch.full((16, 2), scale, device="cuda", dtype=torch.float16)
    zeros = torch.full((16, 2), zero, device="cuda", dtype=torch.uint8)
    d = {"codes": torch.full((16, 32), 0xFF, device="cuda", dtype=torch.uint8), "scales": scales, "zeros": zeros, "bias": None}
    layer = bn.Q4Linear(0, 64, 16, d["codes"], scales, zeros=zeros, group=32, dtype="fp16")
    x = torch.rand(40, 64, device="cuda", generator=gen(1)).half() * 2.0 ** -8
    y = torch.empty(40, 16, device="cuda", dtype=torch.float16)
    layer.run(x, y)
    ref, tol = linear_ref(d, x, 64, 32, "fp16")
    within(y, ref, tol)


def test_layers_beside_a_network_on_another_stream():
    """The linear layer's tensor-memory kernel and the binary network's, at
    once on two streams: each result is that of the call alone."""
    import os

    from oracle_util import synth

    m = bn.Model(os.path.join(os.path.dirname(__file__), "golden", "unet_c8_mixed_s1.blob"))
    patches = torch.from_numpy(synth(7, 0, 8, m.n_bands, 32, 32)).cuda()
    layer, d = linear_case(1, 200, 2048, 1024, 64, "bf16", True, False)
    y0, logits0 = torch.empty(200, 1024, device="cuda", dtype=torch.bfloat16), torch.empty(8, 3, 32, 32, device="cuda")
    layer.run(d["x"], y0)
    m.forward_device(0, patches, 8, 32, 32, logits0)
    torch.cuda.synchronize()
    ys = [torch.empty_like(y0) for _ in range(20)]
    logits = [torch.empty_like(logits0) for _ in range(20)]
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for y, z in zip(ys, logits):
        layer.run(d["x"], y, stream=a)
        m.forward_device(0, patches, 8, 32, 32, z, b.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(y, y0) for y in ys) and all(torch.equal(z, logits0) for z in logits)


FIRST_CALLS = """
import sys
import torch
import bnns_to_c_b200 as bn

def run(eager):
    t, g = torch.bfloat16, torch.Generator(device="cuda").manual_seed(1)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g).to(t)
    whole = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    layers = [bn.Q4Linear(0, k, n, torch.randint(0, 256, (n, k // 2), device="cuda", generator=g, dtype=torch.uint8),
                          rnd(n, k // 64).abs(), group=64) for k, n in ((512, 256), (4096, 64))]
    xs = [rnd(m, l.n_in) for l in layers for m in (1, 12, 300)]
    ys = [torch.zeros(x.shape[0], l.n_out, device="cuda", dtype=t) for l, x in zip([l for l in layers for _ in range(3)], xs)]
    c = bn.KVCache(0, 40, 64, 2, 128, bits=8)
    k, v, q = rnd(900, 2, 128), rnd(900, 2, 128), rnd(3, 16, 128)
    table, pre = torch.arange(30, dtype=torch.int32, device="cuda").view(3, 10), torch.arange(30, 35, dtype=torch.int32, device="cuda")
    start, off, n = whole(0, 0, 0), whole(0, 300, 310, 900), whole(300, 10, 590)
    gk, gv, outs = torch.zeros_like(k), torch.zeros_like(v), [torch.zeros_like(q) for _ in range(2)]
    works = [torch.empty(c.attend_work(3, 16, p), device="cuda", dtype=torch.uint8) for p in (0, 200)]
    def calls(st):
        for i, (x, y) in enumerate(zip(xs, ys)):
            layers[i // 3].run(x, y, stream=st)
        c.write(k, v, table, start, offsets=off, stream=st)
        c.read(gk, gv, table, start, offsets=off, stream=st)
        c.attend(q, n, table, outs[0], works[0], stream=st)
        c.attend(q, n, table, outs[1], works[1], prefix=pre, prefix_tokens=200, stream=st)
    torch.cuda.synchronize()
    if eager:
        calls(torch.cuda.current_stream())
    else:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            calls(torch.cuda.current_stream())
        graph.replay()
    torch.cuda.synchronize()
    return ys + [gk, gv] + outs

captured, eager = run(False), run(True)
assert all(torch.equal(a, b) and a.abs().sum() > 0 for a, b in zip(captured, eager))
assert bn.q4_wait_timeouts(0) == 0
print("same")
"""


@pytest.mark.parametrize("pdl", ["1", "0"])
def test_first_calls_of_a_process_are_captured(pdl):
    """No call needs one before it: the first ones of a process go into a
    graph (with and without programmatic launches)."""
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST_CALLS], cwd=root, env={**os.environ, "BNN_PDL": pdl}, capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "same", r.stdout[-2000:] + r.stderr[-2000:]
