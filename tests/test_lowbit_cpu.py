"""The low-bit operators (include/bnn_lowbit.h) without a GPU: the index
arithmetic that their kernels share, walked under the sanitizers, and the
refusals of every entry point, on handles made without a device."""

import ctypes
import os
import re
import shutil
import subprocess

import numpy as np
import pytest
import torch

import bnns_to_c_b200 as bn

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)


def test_layouts_pages_and_split_under_the_sanitizers(tmp_path):
    cxx = shutil.which("g++")
    if not cxx:
        pytest.skip("no g++")
    exe = str(tmp_path / "lowbit_layout")
    r = subprocess.run([cxx, "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
                        os.path.join(HERE, "san", "lowbit_layout.cpp"), "-o", exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    assert r.stdout.split() == ["linear", "cache", "pages", "split"]


def test_header_functions_are_exported():
    src = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "bnn_lowbit.h")).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(bnn_(?:q4|kv)_\w+)\s*\(", src)))
    assert len(names) == 11
    L = ctypes.CDLL(bn.LIB_PATH)
    assert not [n for n in names if not hasattr(L, n)]


def refused(code, text, fn, *args):
    rc = fn(*args)
    msg = bn.lib().bnn_last_error().decode()
    assert rc == code and re.search(text, msg), (rc, msg)


ARG, CUDA = bn.BNN_ERR_ARG, bn.BNN_ERR_CUDA


# ------------------------------------------------------------------ linear
def q4(device=-1, n_in=64, n_out=16, group=32, type_=0, codes=16, scales=16):
    h = ctypes.c_void_p()
    return bn.lib().bnn_q4_layer_create(device, n_in, n_out, group, type_, codes, scales, None, None, ctypes.byref(h)), h


@pytest.mark.parametrize("kw", [{"n_in": 0}, {"n_in": -5}, {"n_out": 0}, {"n_in": (1 << 24) + 1}, {"group": 0}, {"group": 48},
                                {"group": -32}, {"type_": 2}, {"codes": None}, {"scales": None}, {"device": -2}])
def test_linear_create_refusals(kw):
    rc, h = q4(**kw)
    assert rc == ARG and not h.value


def test_linear_run_refusals():
    rc, h = q4()
    assert rc == 0
    run = bn.lib().bnn_q4_layer_run
    refused(ARG, "bad arguments", run, None, 16, 64, 1, 16, 16, None)
    refused(ARG, "bad arguments", run, h, 16, 64, -1, 16, 16, None)
    refused(ARG, "NULL", run, h, None, 64, 1, 16, 16, None)
    refused(ARG, "NULL", run, h, 16, 64, 1, None, 16, None)
    refused(ARG, "aligned", run, h, 17, 64, 1, 16, 16, None)
    refused(ARG, "strides", run, h, 16, 63, 2, 16, 16, None)
    refused(ARG, "strides", run, h, 16, 64, 2, 16, 15, None)
    refused(ARG, "rows", run, h, 16, 64, (1 << 19) + 1, 16, 16, None)
    refused(CUDA, "without a device", run, h, 16, 0, 1, 16, 0, None)  # one row needs no stride
    refused(CUDA, "without a device", run, h, None, 0, 0, None, 0, None)
    bn.lib().bnn_q4_layer_destroy(h)
    bn.lib().bnn_q4_layer_destroy(None)


def test_linear_binding_checks_its_tensors():
    codes, scales = np.zeros((16, 33), np.uint8), torch.zeros(16, 3, dtype=torch.bfloat16)
    make = lambda **kw: bn.Q4Linear(**{**dict(device=-1, n_in=65, n_out=16, codes=codes, scales=scales, group=32), **kw})  # noqa: E731
    layer = make()
    for kw, text in (({"codes": codes[:, :32]}, "codes: shape"), ({"scales": scales[:8]}, "scales: shape"),
                     ({"scales": scales.half()}, "bfloat16|float16"), ({"codes": codes.astype(np.int32)}, "another size"),
                     ({"zeros": np.zeros((16, 2), np.uint8)}, "zeros: shape"), ({"bias": np.zeros(16)}, "another size"),
                     ({"dtype": "fp32"}, "dtype"), ({"group": 40}, "scales: shape"), ({"n_in": 0}, "inputs"),
                     ({"codes": np.zeros((33, 16), np.uint8).T}, "contiguous")):
        with pytest.raises(bn.BnnError, match=text) as e:
            make(**kw)
        assert e.value.code == ARG
    x, y = torch.zeros(2, 65, dtype=torch.bfloat16), torch.zeros(2, 16, dtype=torch.bfloat16)
    for a, b, text in ((x.half(), y, "x: torch.float16"), (x[:, :64], y, "x: shape"), (x, y[:1], "y: shape"), (x[0], y, "dimensions"),
                       (torch.zeros(65, 2, dtype=torch.bfloat16).T, y, "contiguous"), (np.zeros((2, 65)), y, "a tensor is needed")):
        with pytest.raises(bn.BnnError, match=text) as e:
            layer.run(a, b)
        assert e.value.code == ARG
    with pytest.raises(bn.BnnError) as e:
        layer.run(x, y)
    assert e.value.code == CUDA
    layer.close()
    with pytest.raises(bn.BnnError) as e:  # a closed handle
        layer.run(x, y)
    assert e.value.code == ARG


# ------------------------------------------------------------------ cache
def kv(device=-1, pages=4, pt=32, heads=2, dim=64, bits=8, group=0, type_=0):
    h = ctypes.c_void_p()
    return bn.lib().bnn_kv_cache_create(device, pages, pt, heads, dim, bits, group, type_, ctypes.byref(h)), h


@pytest.mark.parametrize("kw", [{"pages": 0}, {"pages": -1}, {"pt": 8}, {"pt": 48}, {"pt": 512}, {"heads": 0}, {"heads": 4097},
                                {"dim": 0}, {"dim": 60}, {"dim": 264}, {"bits": 2}, {"bits": 16}, {"group": 16}, {"group": 48},
                                {"group": -1}, {"type_": 2}, {"device": -2}])
def test_cache_create_refusals(kw):
    rc, h = kv(**kw)
    assert rc == ARG and not h.value


def test_cache_create_takes_its_whole_range():
    for dim in range(8, 257, 8):
        for group in (0, 32, 64, 128, dim):
            for bits in (4, 8):
                rc, h = kv(dim=dim, group=group, bits=bits)
                assert rc == 0
                groups = -(-dim // (group or dim))
                # codes of a row padded to 64 numbers and 2 bytes a scale, of at most twice as many, keys and values
                least = 2 * 4 * 32 * 2 * (dim * bits // 8 + 2 * groups)
                assert least <= bn.lib().bnn_kv_cache_bytes(h) < 2 * 4 * 32 * 2 * ((dim + 56) * bits // 8 + 4 * groups) + 1024
                bn.lib().bnn_kv_cache_destroy(h)
    bn.lib().bnn_kv_cache_destroy(None)
    assert bn.lib().bnn_kv_cache_bytes(None) == 0


@pytest.mark.parametrize("name", ["write", "read"])
def test_cache_rows_refusals(name):
    _, h = kv()
    fn = getattr(bn.lib(), "bnn_kv_cache_" + name)
    good = dict(h=h, k=16, kt=128, kh=64, v=16, vt=128, vh=64, tokens=5, seqs=2, table=16, width=3, start=16, off=16)
    call = lambda **kw: (fn, *{**good, **kw}.values(), None)  # noqa: E731
    refused(CUDA, "without a device", *call())
    for kw in ({"h": None}, {"tokens": -1}, {"tokens": (1 << 30) + 1}, {"seqs": -1}, {"width": -1}, {"k": None}, {"v": None}, {"table": None}, {"start": None},
               {"k": 17}, {"table": 18}, {"start": 18}, {"off": 18}, {"off": None}):
        refused(ARG, "bnn_kv_cache_" + name, *call(**kw))
    for kw in ({"kt": 1 << 31}, {"vh": -(1 << 31)}):
        refused(ARG, "stride", *call(**kw))
    refused(CUDA, "without a device", *call(off=None, tokens=2))
    refused(CUDA, "without a device", *call(tokens=0, k=None, v=None, table=None))
    for kw in ({"kh": 63}, {"vh": 0}, {"kt": 63}, {"vt": -64}):  # rows that lie over one another: in an output only
        refused(*((CUDA, "without a device") if name == "write" else (ARG, "strides")), *call(**kw))
    bn.lib().bnn_kv_cache_destroy(h)


def test_attend_refusals():
    _, h = kv()
    work = bn.lib().bnn_kv_attend_work
    need = work(h, 3, 8, 0)
    assert need > 0 and work(h, 0, 8, 0) == 0 and work(h, 3, 8, 10) > need
    for bad in ((None, 3, 8, 0), (h, -1, 8, 0), (h, 16385, 8, 0), (h, 3, 7, 0), (h, 3, 0, 0), (h, 3, -2, 0), (h, 3, 8, -1)):
        assert work(*bad) == 0
    good = dict(h=h, q=16, qs=512, qh=64, seqs=3, heads=8, lengths=16, table=16, width=3, prefix=None, pp=0, pt=0, scale=0.125,
                out=16, os=512, oh=64, lse=None, work=16, bytes=need)
    call = lambda **kw: (bn.lib().bnn_kv_attend, *{**good, **kw}.values(), None)  # noqa: E731
    refused(CUDA, "without a device", *call())
    for kw, text in (({"h": None}, "bad"), ({"seqs": -1}, "bad"), ({"seqs": 16385}, "bad"), ({"heads": 7}, "multiple"),
                     ({"heads": 0}, "multiple"), ({"pt": -1}, "bad"), ({"q": None}, "NULL"), ({"out": None}, "NULL"),
                     ({"lengths": None}, "NULL"), ({"table": None}, "NULL"), ({"q": 17}, "aligned"), ({"out": 17}, "aligned"),
                     ({"lse": 18}, "aligned"), ({"lengths": 18}, "aligned"), ({"width": -1}, "negative"), ({"pp": -1}, "negative"),
                     ({"scale": float("nan")}, "finite"), ({"scale": float("inf")}, "finite"), ({"scale": 3e38}, "finite"), ({"work": None}, "workspace"),
                     ({"work": 24}, "workspace"), ({"bytes": need - 1}, "workspace"), ({"oh": 63}, "strides"), ({"os": 0}, "strides"),
                     ({"pt": 33, "pp": 1, "prefix": 16}, "prefix of 33"), ({"pt": 32, "pp": 1, "prefix": None}, "prefix"),
                     ({"width": 1 << 26}, "2\\^31"), ({"seqs": 16384, "width": (1 << 26) - 9, "bytes": 1 << 40}, "too many")):
        refused(ARG, text, *call(**kw))
    refused(CUDA, "without a device", *call(pt=32, pp=1, prefix=16, bytes=work(h, 3, 8, 32)))
    refused(CUDA, "without a device", *call(seqs=0, q=None, out=None, lengths=None, work=None, bytes=0))
    refused(CUDA, "without a device", *call(width=0, table=None))
    bn.lib().bnn_kv_cache_destroy(h)


def test_cache_binding_checks_its_tensors():
    c = bn.KVCache(-1, 4, 32, 2, 64, bits=4, group=32, dtype="fp16")
    half = lambda *s: torch.zeros(*s, dtype=torch.float16)  # noqa: E731
    whole = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    k, table, start, off = half(5, 2, 64), whole(3, 4), whole(3), whole(4)
    for args, text in (((k.float(), k, table, start, off), "k: torch.float32"), ((k, k[:4], table, start, off), "v: shape"),
                       ((k[:, :1], k, table, start, off), "k: shape"), ((k, k, table[:2], start, off), "table: shape"),
                       ((k, k, table.long(), start, off), "table: torch.int64"), ((k, k, table, start, off[:3]), "offsets: shape"),
                       ((k, k, table[:, ::2], start, off), "contiguous"), ((k, k, table, start, None), "need offsets"),
                       ((half(5, 64, 2).transpose(1, 2), k, table, start, off), "contiguous")):
        for fn in (c.write, c.read):
            with pytest.raises(bn.BnnError, match=text) as e:
                fn(*args)
            assert e.value.code == ARG
    with pytest.raises(bn.BnnError) as e:
        c.write(k, k, table, start, off)
    assert e.value.code == CUDA
    q, out, lengths = half(3, 8, 64), half(3, 8, 64), whole(3)
    work = torch.zeros(c.attend_work(3, 8, 40), dtype=torch.uint8)
    for kw, text in (({"d_q": q[:, :7]}, "multiple|shape"), ({"d_out": out[:2]}, "out: shape"), ({"lengths": lengths[:2]}, "lengths: shape"),
                     ({"lse": half(3, 8)}, "lse: torch.float16"), ({"work": work[:100]}, "workspace"),
                     ({"prefix_tokens": 40}, "prefix"), ({"prefix": whole(1), "prefix_tokens": 40}, "prefix of 40"),
                     ({"scale": float("nan")}, "finite"), ({"d_q": q[0]}, "q: .*dimensions")):
        with pytest.raises(bn.BnnError, match=text) as e:
            c.attend(**{**dict(d_q=q, lengths=lengths, table=table, d_out=out, work=work), **kw})
        assert e.value.code == ARG
    with pytest.raises(bn.BnnError, match="multiple"):
        c.attend_work(3, 7)
    with pytest.raises(bn.BnnError) as e:
        c.attend(q, lengths, table, out, work, prefix=whole(2), prefix_tokens=40)
    assert e.value.code == CUDA
    c.close()


def test_create_without_a_gpu_reports_it():
    if torch.cuda.is_available():
        pytest.skip("GPU present")
    rc, h = kv(device=0)
    assert rc == CUDA and not h.value
    buf = np.zeros(4096, np.uint8)
    rc, h = q4(device=0, codes=buf.ctypes.data, scales=buf.ctypes.data)
    assert rc == CUDA and not h.value


def test_dependents_start_behind_the_tensor_memory_allocation():
    """A programmatic dependent that takes tensor memory and waits for the
    grid before it must not start while a CTA of that grid still waits for its
    own: the order in the source of the one kernel that allocates some."""
    src = open(os.path.join(ROOT, "bnns_to_c_b200", "csrc", "q4_linear.cu")).read()
    body = src[src.index("q4_tiles_kernel(const"):]
    alloc, barrier, start = body.index("t5_alloc("), body.index("__syncthreads()"), body.index("grid_launch()")
    assert alloc < barrier < start
    assert src.count("t5_alloc(") == 1


def test_outputs_that_lie_over_one_another_are_refused():
    """Rows and heads that share numbers, although each stride alone is wide
    enough; layouts that only look alike are taken."""
    _, h = kv()
    read = lambda tokens, kt, kh: (bn.lib().bnn_kv_cache_read, h, 16, kt, kh, 16, 128, 64, tokens, 2, 16, 3, 16, 16, None)  # noqa: E731
    other = lambda tokens, vt, vh: (bn.lib().bnn_kv_cache_read, h, 16, 128, 64, 16, vt, vh, tokens, 2, 16, 3, 16, 16, None)  # noqa: E731
    need = bn.lib().bnn_kv_attend_work(h, 3, 8, 0)
    att = lambda os, oh: (bn.lib().bnn_kv_attend, h, 16, 512, 64, 3, 8, 16, 16, 3, None, 0, 0, 0.125, 16, os, oh, None, 16, need, None)  # noqa: E731
    for fn in (read, other):
        for tokens, st, hd in ((5, 64, 64), (2, 64, 64), (5, 64, 256), (5, 100, 64), (5, 64, 319), (5, 65, 130), (9, 127, 64)):
            refused(ARG, "over one another", *fn(tokens, st, hd))
        # heads outside, tokens outside, woven into one another, one token, a gap that just fits
        for tokens, st, hd in ((5, 64, 320), (5, 128, 64), (5, 128, 192), (1, 0, 64), (3, 200, 100), (5, 130, 65), (5, 1 << 30, 1 << 30 | 64)):
            refused(CUDA, "without a device", *fn(tokens, st, hd))
    for st, hd in ((64, 64), (511, 64), (64, 128), (200, 100), (300, 75), (64, 191)):
        refused(ARG, "over one another", *att(st, hd))
    for st, hd in ((512, 64), (64, 192), (128, 448), (1 << 62, 64), (64, 1 << 62)):
        refused(CUDA, "without a device", *att(st, hd))
    bn.lib().bnn_kv_cache_destroy(h)
