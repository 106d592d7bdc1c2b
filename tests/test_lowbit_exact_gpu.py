"""The low-bit operators (include/bnn_lowbit.h) on the GPU on inputs whose
answer is exact, or whose every part shows: a token or an input that is lost,
doubled or weighted wrongly anywhere changes a result by far more than what
is allowed."""

import math

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
    yield
    assert bn.q4_wait_timeouts(0) == 0


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def whole(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------ linear
@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("m,k,n,group", [
    (1, 31, 17, 32), (2, 512, 512, 128), (1, 16384, 64, 128), (8, 8192, 130, 64), (3, 4160, 100, 64), (5, 6464, 300, 32), (1, 7168, 600, 256),
    (9, 1030, 77, 32), (16, 9000, 300, 64), (16, 4096, 2048, 64), (12, 3200, 100, 32), (16, 4096, 4096, 128), (33, 2704, 90, 128),
    (64, 640, 300, 64), (70, 3200, 100, 32), (129, 448, 128, 64), (200, 1800, 130, 64), (128, 5001, 130, 64), (40, 4099, 200, 32),
    (260, 4098, 300, 128), (700, 2704, 1000, 64), (2048, 1024, 512, 128), (1000, 3001, 1111, 64)])
def test_linear_sums_without_any_rounding(m, k, n, group, kind):
    """x of -1, 0 and 1, scales that are powers of two: weights, products and
    sums are exact in any order, so the result is the exact one, rounded."""
    g, t = gen(m + k), TYPES[kind]
    ng = -(-k // group)
    x = torch.randint(-1, 2, (m, k), device="cuda", generator=g).to(t)
    codes = torch.randint(0, 256, (n, (k + 1) // 2), device="cuda", generator=g, dtype=torch.uint8)
    scales = torch.exp2(-torch.randint(0, 4, (n, ng), device="cuda", generator=g).float()).to(t)
    zeros = torch.randint(0, 16, (n, ng), device="cuda", generator=g, dtype=torch.uint8)
    bias = torch.randint(-64, 65, (n,), device="cuda", generator=g).float() / 8
    layer = bn.Q4Linear(0, k, n, codes, scales, zeros=zeros, bias=bias, group=group, dtype=kind)
    y = torch.empty(m, n, device="cuda", dtype=t)
    layer.run(x, y)
    q = torch.stack((codes & 15, codes >> 4), -1).flatten(1)[:, :k].double()
    of = torch.arange(k, device="cuda") // group
    w = (q - zeros.double()[:, of]) * scales.double()[:, of]
    ref = x.double() @ w.T + bias.double()
    assert ref.abs().max() < 2 ** 14 and torch.equal(ref * 8, (ref * 8).round())
    assert torch.equal(y, ref.to(t))


# ------------------------------------------------------------------ attention
def cache_of(k, v, bits, group, kind, page, cut):
    """A cache of these tokens in shuffled pages, the first `cut` of them as a
    prefix: (cache, table, prefix pages)."""
    n, heads, dim = k.shape
    n_pre, n_own = -(-cut // page), max(1, -(-(n - cut) // page))
    c = bn.KVCache(0, n_pre + n_own + 3, page, heads, dim, bits=bits, group=group, dtype=kind)
    order = torch.randperm(n_pre + n_own + 3, device="cuda", generator=gen(n)).to(torch.int32)
    pre, own = order[:n_pre].contiguous(), order[n_pre:n_pre + n_own][None].contiguous()
    if cut:
        c.write(k[:cut], v[:cut], pre[None], whole(0), offsets=whole(0, cut))
    c.write(k[cut:], v[cut:], own, whole(0), offsets=whole(0, n - cut))
    return c, own, pre


def attend(c, q, n, own, pre, cut):
    out, lse = torch.full_like(q, 3.0), torch.full(q.shape[:2], 3.0, device="cuda")
    seqs = q.shape[0]
    work = torch.full((c.attend_work(seqs, q.shape[1], cut),), 0xFF, device="cuda", dtype=torch.uint8)
    c.attend(q, torch.full((seqs,), n - cut, dtype=torch.int32, device="cuda"), own.repeat(seqs, 1), out, work, lse=lse, scale=1.0,
             prefix=pre if cut else None, prefix_tokens=cut)
    return out, lse


SHAPES = [(1, 1, 4, 64, 8, 0, 16), (777, 2, 4, 64, 4, 32, 16), (20011, 1, 8, 128, 8, 0, 64), (20011, 8, 8, 128, 8, 0, 64),
          (20011, 2, 16, 128, 4, 32, 64), (9001, 2, 32, 64, 8, 32, 32), (5003, 1, 5, 256, 4, 64, 128), (30000, 3, 2, 192, 8, 64, 256),
          (100003, 2, 4, 128, 8, 128, 64)]


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("n,heads,share,dim,bits,group,page", SHAPES)
@pytest.mark.parametrize("prefix", [False, True])
def test_attend_counts_every_token(n, heads, share, dim, bits, group, page, prefix, kind):
    """All weights are equal (q = 0), and each token has one channel with a
    value of its own group's scale 1, the others 0: a channel's result is the
    number of its tokens over n, the log-sum ln n. Weights, codes and sums are
    exact; 2^-20 for the joins, and a rounding to the type."""
    cut = n * 2 // 3 if prefix else 0
    top = 2 ** (bits - 1) - 1
    at = (torch.arange(n, device="cuda") * 7) % dim
    v = torch.zeros(n, heads, dim, device="cuda")
    v[torch.arange(n, device="cuda"), :, at] = float(top)
    k = torch.randn(n, heads, dim, device="cuda", generator=gen(1))
    c, own, pre = cache_of(k.to(TYPES[kind]), v.to(TYPES[kind]), bits, group, kind, page, cut)
    q = torch.zeros(2, heads * share, dim, device="cuda", dtype=TYPES[kind])
    out, lse = attend(c, q, n, own, pre, cut)
    ref = torch.bincount(at, minlength=dim).double() * top / n
    tol = ref * (torch.finfo(TYPES[kind]).eps / 2 + 2.0 ** -20)
    assert ((out.double() - ref).abs() <= tol).all()
    assert ((lse.double() - math.log(n)).abs() <= 2.0 ** -20 + 4 * U * math.log(n)).all()


@pytest.mark.parametrize("n,heads,share,dim,bits,group,page", SHAPES)
@pytest.mark.parametrize("prefix", [False, True])
def test_attend_finds_each_position(n, heads, share, dim, bits, group, page, prefix):
    """Keys spell their position in 17 channels of +-1, queries the position
    they want, 96 nats above every other: the result is that token's value as
    the cache holds it, bit for bit. Positions at the borders of steps, blocks,
    pages and the prefix, and others at random."""
    kind, cut = "bf16", n * 2 // 3 if prefix else 0
    bit = torch.arange(17, device="cuda")
    spell = lambda p: ((p[..., None] >> bit) & 1) * 2.0 - 1.0  # noqa: E731
    k = torch.zeros(n, heads, dim, device="cuda")
    k[:, :, :17] = spell(torch.arange(n, device="cuda"))[:, None]
    v = torch.randn(n, heads, dim, device="cuda", generator=gen(2)).to(TYPES[kind])
    c, own, pre = cache_of(k.to(TYPES[kind]), v, bits, group, kind, page, cut)
    held = torch.empty_like(v)
    if cut:
        c.read(torch.empty_like(v[:cut]), held[:cut], pre[None], whole(0), offsets=whole(0, cut))
    c.read(torch.empty_like(v[cut:]), held[cut:], own, whole(0), offsets=whole(0, n - cut))
    want = {0, n - 1, cut, max(0, cut - 1)}
    for step in (16, 32, 64, 256, page, 1024, 4096):
        for base in (0, cut, n // 2 // step * step):
            want |= {base + step - 1, base + step, base + 2 * step - 1}
    want = torch.tensor(sorted(p for p in want if p < n), device="cuda")
    seqs = -(-want.numel() // (heads * share)) + 1
    fill = torch.randint(0, n, (seqs * heads * share,), device="cuda", generator=gen(3))
    fill[: want.numel()] = want
    fill = fill[torch.randperm(fill.numel(), device="cuda", generator=gen(4))].view(seqs, heads * share)
    q = torch.zeros(seqs, heads * share, dim, device="cuda")
    q[:, :, :17] = spell(fill) * 48.0
    out, _ = attend(c, q.to(TYPES[kind]), n, own, pre, cut)
    of = torch.arange(heads * share, device="cuda") // share
    assert torch.equal(out, held[fill, of[None].expand_as(fill)])


# ------------------------------------------------------------------ streams joined by events
@pytest.mark.parametrize("captured", [False, True])
def test_calls_behind_another_streams_event(captured):
    """Each call starts early behind the one before it in its stream, but not
    before what its stream waits for: inputs that a second stream writes late,
    behind an event, while the first stream's last kernel allows early starts."""
    t = torch.bfloat16
    layer = bn.Q4Linear(0, 512, 256, torch.randint(0, 256, (256, 256), device="cuda", generator=gen(1), dtype=torch.uint8),
                        torch.ones(256, 8, device="cuda", dtype=t), group=64)
    c = bn.KVCache(0, 4, 64, 2, 128, bits=8)
    table, start, n = whole(0, 1, 2, 3).view(1, 4), whole(0), whole(200)
    off = whole(0, 200)
    src = {"x": torch.randn(40, 512, device="cuda", generator=gen(2)).to(t), "q": torch.randn(1, 8, 128, device="cuda", generator=gen(3)).to(t),
           "k": torch.randn(200, 2, 128, device="cuda", generator=gen(4)).to(t), "v": torch.randn(200, 2, 128, device="cuda", generator=gen(5)).to(t)}
    late = {k: torch.zeros_like(v) for k, v in src.items()}
    warm = torch.zeros(3, 512, device="cuda", dtype=t)
    y0, ys = torch.empty(3, 256, device="cuda", dtype=t), [torch.empty(m, 256, device="cuda", dtype=t) for m in (3, 12, 40)]
    gk, gv, out = torch.empty_like(src["k"]), torch.empty_like(src["v"]), torch.empty_like(src["q"])
    work = torch.empty(c.attend_work(1, 8), device="cuda", dtype=torch.uint8)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()

    def run():
        """Every call on a, right behind a short kernel of a and an event of b."""
        calls = [(("x",), lambda m=m, y=y: layer.run(late["x"][:m], y, stream=a)) for m, y in zip((3, 12, 40), ys)]
        calls += [(("k", "v"), lambda: c.write(late["k"], late["v"], table, start, offsets=off, stream=a)),
                  ((), lambda: c.read(gk, gv, table, start, offsets=off, stream=a)),
                  (("q",), lambda: c.attend(late["q"], n, table, out, work, stream=a))]
        for names, call in calls:
            b.wait_stream(a)
            with torch.cuda.stream(b):
                torch.cuda._sleep(400_000)  # 0.2 ms
                for k in names:
                    late[k].copy_(src[k])
            layer.run(warm, y0, stream=a)
            a.wait_stream(b)
            call()

    torch.cuda.synchronize()
    if captured:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=a):
            run()
    for _ in range(3):
        for v in late.values():
            v.zero_()
        torch.cuda.synchronize()
        g.replay() if captured else run()
        torch.cuda.synchronize()
        got = [x.clone() for x in ys + [gk, gv, out]]
        for m, y in zip((3, 12, 40), ys):
            layer.run(src["x"][:m], y)
        c.write(src["k"], src["v"], table, start, offsets=off)
        c.read(gk, gv, table, start, offsets=off)
        c.attend(src["q"], n, table, out, work)
        torch.cuda.synchronize()
        assert all(torch.equal(x, z) for x, z in zip(got, ys + [gk, gv, out]))
        assert got[2].abs().sum() > 0 and got[5].abs().sum() > 0


# ------------------------------------------------------------------ the ends of the documented ranges
@pytest.mark.parametrize("heavy", [False, True])
def test_linear_most_rows(heavy):
    """2^19 rows, the most of a call; heavy: with weights outside fp16."""
    m, k, n = 1 << 19, 64, 40
    x = torch.randint(-1, 2, (m, k), device="cuda", generator=gen(1)).half()
    codes = torch.randint(0, 256, (n, k // 2), device="cuda", generator=gen(2), dtype=torch.uint8)
    scales = torch.full((n, 2), 0.25, device="cuda", dtype=torch.float16)
    if heavy:
        zeros = torch.full((n, 2), 8, device="cuda", dtype=torch.uint8)
        scales[7], codes[7], zeros[7, 0] = 8192.0, 0x8F, 0  # weights 15 * 8192 and 8 * 8192, then 7 * 8192 and 0
        x[:, :32] = 0.0
        x[:, 32::2] = torch.where(torch.arange(16, device="cuda") == 3, x[:, 32::2], 0.0)  # one of them in each sum
    else:
        zeros = None
    layer = bn.Q4Linear(0, k, n, codes, scales, zeros=zeros, group=32, dtype="fp16")
    y = torch.empty(m, n, device="cuda", dtype=torch.float16)
    layer.run(x, y)
    q = torch.stack((codes & 15, codes >> 4), -1).flatten(1).float()
    z = zeros.float().repeat_interleave(32, 1) if heavy else 8.0
    w = (q - z) * scales.float().repeat_interleave(32, 1)
    assert (w.abs().max() > 65504) == heavy
    ref = x.float() @ w.T  # exact: whole multiples of a quarter below 2^24 of them
    assert torch.equal(y, ref.half())


def test_cache_most_heads():
    """4096 kv heads, written and read back; a group wider than the head."""
    for dim, bits, group in ((8, 8, 32), (16, 4, 0)):
        c = bn.KVCache(0, 3, 16, 4096, dim, bits=bits, group=group)
        top = 2 ** (bits - 1) - 1
        x = [torch.randint(-top, top + 1, (37, 4096, dim), device="cuda", generator=gen(i)).float() for i in (1, 2)]
        for v in x:
            v[..., 0] = top  # scale 1: every code is held exactly
        x = [v.to(torch.bfloat16) for v in x]
        table, off = whole(2, 0, 1)[None], whole(0, 37)
        c.write(*x, table, whole(5), offsets=off)
        got = [torch.zeros_like(v) for v in x]
        c.read(*got, table, whole(5), offsets=off)
        assert all(torch.equal(a, b) for a, b in zip(x, got))


def counted(n, heads, dim, kind):
    """Values with 127 in one channel a token, keys of any kind."""
    at = (torch.arange(n, device="cuda") * 7) % dim
    v = torch.zeros(n, heads, dim, device="cuda")
    v[torch.arange(n, device="cuda"), :, at] = 127.0
    return torch.randn(n, heads, dim, device="cuda", generator=gen(1)).to(kind), v.to(kind), torch.nn.functional.one_hot(at, dim).double() * 127


@pytest.mark.parametrize("prefix", [0, 50])
@pytest.mark.parametrize("dim,share", [(64, 2), (256, 9)])
def test_attend_most_sequences(dim, share, prefix):
    """16384 sequences, the most of a call, of 0 to 70 tokens, all in the same
    pages; every weight is the same."""
    seqs, n = 16384, 70
    k, v, one = counted(n + prefix, 1, dim, torch.float16)
    c = bn.KVCache(0, 9, 16, 1, dim, bits=8, dtype="fp16")
    own, pre = whole(0, 1, 2, 3, 4), whole(5, 6, 7, 8)
    c.write(k[prefix:], v[prefix:], own[None], whole(0), offsets=whole(0, n))
    if prefix:
        c.write(k[:prefix], v[:prefix], pre[None], whole(0), offsets=whole(0, prefix))
    lengths = torch.randint(0, n + 1, (seqs,), device="cuda", generator=gen(2), dtype=torch.int32)
    q, out = torch.zeros(seqs, share, dim, device="cuda", dtype=torch.float16), torch.full((seqs, share, dim), 3.0, device="cuda", dtype=torch.float16)
    lse = torch.full((seqs, share), 3.0, device="cuda")
    work = torch.full((c.attend_work(seqs, share, prefix),), 0xFF, device="cuda", dtype=torch.uint8)
    c.attend(q, lengths, own[None].repeat(seqs, 1), out, work, lse=lse, prefix=pre if prefix else None, prefix_tokens=prefix)
    sums = torch.cat((torch.zeros(1, dim, device="cuda", dtype=torch.float64), one[prefix:].cumsum(0))) + one[:prefix].sum(0)
    count = (lengths + prefix).double()
    ref = (sums[lengths.long()] / count.clamp(min=1)[:, None])[:, None].expand(-1, share, -1)
    assert ((out.double() - ref).abs() <= ref * (2.0 ** -11 + 2.0 ** -20)).all()
    want = count.log()[:, None].expand(-1, share)
    near = (lse.double() - want).abs() <= 2.0 ** -20 + 4 * U * want.abs()
    assert (near | ((lse == want) & (count == 0)[:, None])).all()


@pytest.mark.parametrize("prefix", [0, 40])
def test_attend_most_query_heads(prefix):
    """65536 query heads of one kv head, the most of a call."""
    dim, n, heads = 64, 300, 65536
    k, v, one = counted(n + prefix, 1, dim, torch.bfloat16)
    c = bn.KVCache(0, 22, 16, 1, dim, bits=8)
    own, pre = torch.arange(19, device="cuda", dtype=torch.int32), whole(19, 20, 21)
    c.write(k[prefix:], v[prefix:], own[None], whole(0), offsets=whole(0, n))
    if prefix:
        c.write(k[:prefix], v[:prefix], pre[None], whole(0), offsets=whole(0, prefix))
    q, out = torch.zeros(1, heads, dim, device="cuda", dtype=torch.bfloat16), torch.full((1, heads, dim), 3.0, device="cuda", dtype=torch.bfloat16)
    lse = torch.full((1, heads), 3.0, device="cuda")
    work = torch.full((c.attend_work(1, heads, prefix),), 0xFF, device="cuda", dtype=torch.uint8)
    c.attend(q, whole(n), own[None], out, work, lse=lse, prefix=pre if prefix else None, prefix_tokens=prefix)
    ref = one.sum(0) / (n + prefix)
    assert ((out.double() - ref).abs() <= ref * (2.0 ** -8 + 2.0 ** -20)).all()
    assert ((lse.double() - math.log(n + prefix)).abs() <= 2.0 ** -20 + 4 * U * math.log(n + prefix)).all()
