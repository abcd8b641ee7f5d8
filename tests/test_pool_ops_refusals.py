"""What the operators over the fp16 page pool refuse, and that they do so before any device work: the C entries and
their Python twin over a device that only counts launches (tests/native/fake_device.cpp, fake_pool.cpp), no GPU needed."""
import ctypes as C
import os
import shutil
import subprocess

import numpy as np
import pytest

from rstr import configs, hip
from test_device_ops_refusals import Bare, Dev, inside, ints, refused

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "pretrained-rstr_amd", "csrc")
NEW = [n for n in hip.EXPORTS if n.startswith(("rstr_pool_device", "rstr_pool_rope", "rstr_pool_attn", "rstr_bounds", "rstr_select"))]
BASE = ["rstr_session_open", "rstr_session_close", "rstr_last_error", "rstr_open_error", "rstr_model_bind_synthetic", "rstr_model_close",
        "rstr_pool_open", "rstr_pool_close"]

pytestmark = pytest.mark.skipif(shutil.which("hipcc") is None, reason="no hipcc")


@pytest.fixture(scope="module")
def fake_lib(tmp_path_factory):
    tmp = tmp_path_factory.mktemp("fake")
    so = str(tmp / "librstr_fake_pool.so")
    objects = []
    for src in (os.path.join(CSRC, "pool_ops.cpp"), os.path.join(HERE, "native", "fake_device.cpp"), os.path.join(HERE, "native", "fake_pool.cpp")):
        objects.append(str(tmp / (os.path.basename(src) + ".o")))
        subprocess.run(["hipcc", "-x", "hip", "--offload-arch=gfx950", "--cuda-host-only", "-std=c++17", "-O1", "-w", "-fPIC",
                        "-c", src, "-o", objects[-1]], check=True, capture_output=True, timeout=300)
    subprocess.run(["g++", "-shared", "-Wl,-Bsymbolic", *objects, "-o", so], check=True, capture_output=True, timeout=120)
    real, fake = hip.lib(), C.CDLL(so)
    for n in NEW + BASE:
        f, r = getattr(fake, n), getattr(real, n)
        f.restype, f.argtypes = r.restype, r.argtypes
    fake.fake_stream.restype = C.c_void_p
    return fake


@pytest.fixture
def dev(fake_lib, monkeypatch):
    monkeypatch.setattr(hip, "_lib", fake_lib)
    return fake_lib


def pool(s, n_layers=2, n_kv=2, hd=128, page=16, pages=4):
    cfg = dict(configs.TINY_LLAMA)
    cfg.update(n_layers=n_layers, n_q=n_kv, n_kv=n_kv, head_dim=hd)
    return hip.Pool(hip.Model(s, cfg, seed=1), page, pages)


def test_null_handles(dev):
    for name in NEW:
        f = getattr(dev, name)
        if name.endswith("_close"):
            assert f(None) == 0
        else:
            args = [None if t is C.c_void_p or isinstance(t, type(C.POINTER(C.c_void_p))) else 0 for t in f.argtypes]
            assert f(*args) == -1, name


def test_handles(dev):
    blocks = dev.fake_blocks()
    with hip.Session(0) as s:
        p = pool(s)
        for n_q in (0, 3, -2):
            with pytest.raises(hip.RstrError, match="query heads"):
                hip.PagedAttention(p, n_q, 2, 5)
        for args in ((4, 0, 5), (4, 2, 0), (4, -1, 5)):
            with pytest.raises(hip.RstrError, match="extents"):
                hip.PagedAttention(p, *args)
        for args in ((4, 1 << 23, 1 << 23), (64, 1, 1 << 26), (2, 1, 1 << 24)):
            with pytest.raises(hip.RstrError, match="too many rows"):
                hip.PagedAttention(p, *args)
        hip.PagedAttention(p, 4, 1 << 20, 1 << 20).close()
        b = hip.BlockBounds(p)
        for n_q in (0, 3):
            with pytest.raises(hip.RstrError, match="query heads"):
                hip.BlockSelect(b, n_q, 2, 5, 7)
        for args in ((4, 0, 5, 7), (4, 2, 0, 7), (4, 2, 5, 0)):
            with pytest.raises(hip.RstrError, match="extents"):
                hip.BlockSelect(b, *args)
        for args in ((4, 1, 1 << 23, 1), (4, 1, 1 << 20, 1 << 20)):
            with pytest.raises(hip.RstrError, match="too many rows or pages"):
                hip.BlockSelect(b, *args)
        plan, sel = hip.PagedAttention(p, 4, 2, 5), hip.BlockSelect(b, 4, 2, 5, 7)
        for x, match in ((p, "open attention plans or block bounds"), (b, "open selections")):
            with pytest.raises(hip.RstrError, match=match) as e:
                x.close()
            assert e.value.code == -4
        dev.fake_fail_alloc(1)
        try:
            for f in (lambda: hip.PagedAttention(p, 4, 2, 5), lambda: hip.BlockBounds(p), lambda: hip.BlockSelect(b, 4, 2, 5, 7)):
                with pytest.raises(hip.RstrError) as e:
                    f()
                assert e.value.code == -3
        finally:
            dev.fake_fail_alloc(0)
        sel.close()
        sel.close()
        b.close()
        plan.close()
        p.close()
        q = pool(s)  # a session closes what is open on it, in order
        hip.BlockSelect(hip.BlockBounds(q), 4, 2, 5, 7)
        hip.PagedAttention(q, 4, 2, 5)
    assert dev.fake_blocks() == blocks


def test_views(dev):
    with hip.Session(0) as s:
        p = pool(s)
        k, v = p.pages_device(0, 1), p.pages_device(1, 1)
        assert k.shape == (4, 16, 2, 128) and k.dtype == "float16" and k.data_ptr() != v.data_ptr()
        b = hip.BlockBounds(p)
        assert b.device(1).shape == (4, 2, 2, 128) and b.device(1).data_ptr() - b.device(0).data_ptr() == 4 * 2 * 2 * 128 * 2
        for f, match in ((lambda: p.pages_device(2, 0), "slab or layer"), (lambda: p.pages_device(0, 2), "slab or layer"),
                         (lambda: p.pages_device(0, -1), "slab or layer"), (lambda: b.device(2), "layer"), (lambda: b.device(-1), "layer")):
            refused(dev, hip.RstrError, match, f)


def test_rope_append(dev):
    with hip.Session(0) as s:
        p = pool(s)
        base = dict(layer=0, k=Dev((3, 2, 128)), v=Dev((3, 2, 128)), slots=ints(3), positions=ints(3), frequencies=Dev((64,), "float64"),
                    q=Dev((3, 4, 128)), q_out=Dev((3, 4, 128)))

        def op(**kw):
            p.rope_append(**{**base, **kw}, stream=7)

        op()
        assert dev.fake_stream() == 7
        op(q=None, q_out=None)
        op(frequencies=None, positions=None)
        op(q_gain=Dev((128,)), k_gain=Dev((128,)), eps=0.0, gain_offset=1.0)
        op(frequencies=Dev((8,), "float64"))
        op(q_out=None)                      # in place
        op(q_out=base["q"])
        for match, kw in (("layer", dict(layer=2)), ("layer", dict(layer=-1)), ("rotary dim", dict(frequencies=Dev((72,), "float64"))),
                          ("rotary dim", dict(frequencies=Dev((4,), "float64"))), ("epsilon", dict(q_gain=Dev((128,)), eps=float("nan"))),
                          ("epsilon", dict(k_gain=Dev((128,)), eps=-1.0)), ("epsilon", dict(k_gain=Dev((128,)), gain_offset=float("inf"))),
                          ("aligned", dict(k=Dev((3, 2, 128), shift=2))), ("aligned", dict(slots=ints(3, shift=1))), ("aligned", dict(positions=ints(3, shift=2))),
                          ("aligned", dict(frequencies=Dev((64,), "float64", shift=4))), ("aligned", dict(q_gain=Dev((128,), shift=2))),
                          ("strides", dict(v=Dev((3, 2, 128), strides=(-256, 128, 1)))),
                          ("share elements", dict(q_out=Dev((3, 4, 128), strides=(128, 128, 1))))):
            refused(dev, hip.RstrError, match, lambda: op(**kw))
        for match, kw in (("shape", dict(k=Dev((3, 3, 128)))), ("shape", dict(v=Dev((4, 2, 128)))), ("shape", dict(q=Dev((2, 4, 128)))),
                          ("shape", dict(q_out=Dev((3, 5, 128)))), ("same element type", dict(v=Dev((3, 2, 128), "float16"))),
                          ("same element type", dict(q_out=Dev((3, 4, 128), "float16"))),
                          ("same element type", dict(q=Dev((3, 4, 128), "float16"), q_out=None)), ("without q", dict(q=None)),
                          ("without positions", dict(positions=None)), ("float64", dict(frequencies=Dev((64,)))), ("int32", dict(slots=Dev((3,), "int64"))),
                          ("shape", dict(positions=ints(4))), ("shape", dict(k_gain=Dev((64,)))), ("float32", dict(q_gain=Dev((128,), "float16"))),
                          ("last dimension", dict(k=Dev((3, 2, 128), strides=(512, 256, 2)))), ("session's GPU", dict(q=Dev((3, 4, 128), device=1), q_out=None)),
                          ("float32, float16 or bfloat16", dict(k=Dev((3, 2, 128), "float64")))):
            refused(dev, ValueError, match, lambda: op(**kw))
        n = dev.fake_launches()
        op(k=Dev((0, 2, 128)), v=Dev((0, 2, 128)), slots=ints(0), positions=ints(0), q=Dev((0, 4, 128)), q_out=Dev((0, 4, 128)))
        assert dev.fake_launches() == n


def test_rope_append_of_one_array(dev):
    """Heads of one row as views: apart where their places in the row are; other queries, keys, values and tables are not written into."""
    with hip.Session(0) as s:
        p = pool(s)
        one = Dev((3, 8 * 128))
        view = lambda h, at, row=1024: inside(Dev((3, h, 128), strides=(row, 128, 1)), one, 4 * at)  # noqa: E731
        sl = ints(3)
        p.rope_append(0, view(2, 512), view(2, 768), sl, q=view(4, 0))
        p.rope_append(0, view(2, 0), view(2, 256), sl, q=view(4, 512))
        p.rope_append(0, view(2, 512), view(2, 768), sl, q=Dev((3, 4, 128)), q_out=view(4, 0))
        for k, v, q, out, match in ((view(2, 384), view(2, 768), view(4, 0), None, "overlaps the keys"), (view(2, 512), view(2, 510), view(4, 0), None, "overlaps the keys"),
                                    (view(2, 512), view(2, 768, 1025), view(4, 0), None, "overlaps the keys"),
                                    (Dev((3, 2, 128)), Dev((3, 2, 128)), view(4, 0), view(4, 128), "other queries"),
                                    (Dev((3, 2, 128)), Dev((3, 2, 128)), view(4, 0), view(4, 0, 1023), "other queries")):
            refused(dev, hip.RstrError, match, lambda: p.rope_append(0, k, v, sl, q=q, q_out=out))
        k, out = Dev((3, 2, 128)), Dev((3, 4, 128))
        last = 4 * (3 * 4 * 128 - 1)
        for kw in (dict(slots=inside(ints(3), out, last)), dict(positions=inside(ints(3), out, last)), dict(frequencies=inside(Dev((64,), "float64"), out, last - 4)),
                   dict(q_gain=inside(Dev((128,)), out, last)), dict(k_gain=inside(Dev((128,)), out, last))):
            a = {**dict(slots=sl, positions=ints(3), frequencies=Dev((64,), "float64")), **kw}
            refused(dev, hip.RstrError, "overlaps the call's tables", lambda: p.rope_append(0, k, k, q=Dev((3, 4, 128)), q_out=out, **a))

        class Page(Dev):  # rows of the pool's own pages
            def __init__(self, slab, layer, heads):
                super().__init__((3, heads, 128), "float16")
                self._at = p.pages_device(slab, layer).data_ptr()

            def data_ptr(self):
                return self._at

        h = lambda n: Dev((3, n, 128), "float16")  # noqa: E731
        for slab in (0, 1):
            for a in ((Page(slab, 1, 2), h(2), None, None), (h(2), Page(slab, 1, 2), None, None), (h(2), h(2), Page(slab, 1, 4), h(4)),
                      (h(2), h(2), h(4), Page(slab, 1, 4))):
                refused(dev, hip.RstrError, "layer's pages", lambda: p.rope_append(1, a[0], a[1], sl, q=a[2], q_out=a[3]))
        p.rope_append(0, Page(0, 1, 2), h(2), sl)  # another layer's may be read


def test_attention(dev):
    with hip.Session(0) as s:
        p = pool(s)
        plan = hip.PagedAttention(p, 4, 2, 5)

        def run(**kw):
            a = {**dict(layer=0, q=Dev((5, 4, 128)), ro=ints(3), pt=ints((2, 7)), ln=ints(2), out=Dev((5, 4, 128))), **kw}
            plan.run(*[a.pop(n) for n in ("layer", "q", "ro", "pt", "ln", "out")], **a)

        run()
        run(stream=hip.SESSION_STREAM)
        assert dev.fake_stream() == 0x5e55
        run(max_rows=3, window=4, scale=0.5, blocks=ints((5, 2, 3)))
        for match, kw in (("layer", dict(layer=2)), ("window", dict(window=-1)), ("scale", dict(scale=float("nan"))), ("scale", dict(scale=float("inf"))),
                          ("rows per sequence", dict(max_rows=0)), ("rows per sequence", dict(max_rows=6)),
                          ("batch exceeds", dict(ro=ints(4), ln=ints(3), pt=ints((3, 7)))),
                          ("rows exceed", dict(q=Dev((6, 4, 128)), out=Dev((6, 4, 128)))), ("blocks per row", dict(blocks=ints((5, 2, 0)))),
                          ("width", dict(pt=ints((2, 0)))), ("share elements", dict(out=Dev((5, 4, 128), strides=(128, 128, 1)))),
                          ("aligned", dict(blocks=ints((5, 2, 3), shift=2))),
                          ("aligned", dict(q=Dev((5, 4, 128), "float16", shift=1), out=Dev((5, 4, 128), "float16")))):
            refused(dev, hip.RstrError, match, lambda: run(**kw))
        for match, kw in (("shape", dict(q=Dev((5, 3, 128)))), ("shape", dict(out=Dev((4, 4, 128)))),
                          ("same element type", dict(out=Dev((5, 4, 128), "float16"))), ("shape", dict(ro=ints(4))),
                          ("shape", dict(pt=ints((3, 7)))), ("int32", dict(ln=Dev((2,), "float32"))), ("shape", dict(blocks=ints((4, 2, 3)))),
                          ("shape", dict(blocks=ints((5, 4, 3)))), ("int32", dict(blocks=Dev((5, 2, 3), "int64"))),
                          ("contiguous", dict(blocks=ints((5, 2, 3), strides=(12, 6, 2)))),
                          ("contiguous", dict(pt=ints((2, 7), strides=(14, 1)))), ("session's GPU", dict(pt=ints((2, 7), device=3)))):
            refused(dev, ValueError, match, lambda: run(**kw))
        x = Dev((5, 4, 128))
        refused(dev, hip.RstrError, "overlaps the queries", lambda: run(q=x, out=x))
        for name, a in (("ro", ints(3)), ("pt", ints((2, 7))), ("ln", ints(2)), ("blocks", ints((5, 2, 3)))):
            refused(dev, hip.RstrError, "overlaps the sequences' tables", lambda: run(out=x, **{name: inside(a, x, 4 * (5 * 4 * 128 - 1))}))
            run(out=x, **{name: inside(a, x, 4 * 5 * 4 * 128)})
        n = dev.fake_launches()
        run(q=Dev((0, 4, 128)), out=Dev((0, 4, 128)))
        run(ro=ints(1), ln=ints(0), pt=ints((0, 7)))
        assert dev.fake_launches() == n


def test_bounds_and_selection(dev):
    with hip.Session(0) as s:
        b = hip.BlockBounds(pool(s))
        up = lambda layer=0, ro=ints(3), pt=ints((2, 7)), ln=ints(2), rows=5: b.update(layer, ro, pt, ln, rows, stream=3)  # noqa: E731
        up()
        assert dev.fake_stream() == 3
        for match, kw in (("layer", dict(layer=2)), ("counts", dict(rows=-1)), ("width", dict(pt=ints((2, 0)))), ("too many rows", dict(rows=1 << 25)),
                          ("aligned", dict(ln=ints(2, shift=1)))):
            refused(dev, hip.RstrError, match, lambda: up(**kw))
        for kw in (dict(ro=ints(2)), dict(pt=ints((3, 7)))):
            refused(dev, ValueError, "shape", lambda: up(**kw))
        sel = hip.BlockSelect(b, 4, 2, 5, 7)

        def run(**kw):
            a = {**dict(layer=0, q=Dev((5, 4, 128)), ro=ints(3), pt=ints((2, 7)), ln=ints(2), blocks=ints((5, 2, 3))), **kw}
            sel.run(*[a.pop(n) for n in ("layer", "q", "ro", "pt", "ln", "blocks")], **a)

        run()
        run(first=0, last=3)
        for match, kw in (("layer", dict(layer=2)), ("fit in the list", dict(first=-1)), ("fit in the list", dict(last=0)),
                          ("fit in the list", dict(first=2, last=2)), ("fit in the list", dict(first=2 ** 31 - 1, last=2 ** 31 - 1)),
                          ("blocks per row", dict(blocks=ints((5, 2, 0)))), ("wider", dict(pt=ints((2, 8)))), ("width", dict(pt=ints((2, 0)))),
                          ("batch exceeds", dict(ro=ints(4), ln=ints(3), pt=ints((3, 7)))),
                          ("rows exceed", dict(q=Dev((6, 4, 128)), blocks=ints((6, 2, 3)))), ("aligned", dict(q=Dev((5, 4, 128), shift=1)))):
            refused(dev, hip.RstrError, match, lambda: run(**kw))
        for match, kw in (("shape", dict(q=Dev((5, 3, 128)))), ("shape", dict(blocks=ints((5, 3, 3)))), ("shape", dict(blocks=ints((4, 2, 3)))),
                          ("int32", dict(blocks=Dev((5, 2, 3), "int64"))), ("session's GPU", dict(q=Dev((5, 4, 128), device=1)))):
            refused(dev, ValueError, match, lambda: run(**kw))
        x = ints((5, 2, 3))
        for name, a in (("ro", ints(3)), ("pt", ints((2, 7))), ("ln", ints(2))):
            refused(dev, hip.RstrError, "overlap the sequences' tables", lambda: run(blocks=x, **{name: inside(a, x, 4 * 29)}))
            run(blocks=x, **{name: inside(a, x, 4 * 30)})
        x = ints((5, 2, 3))
        x.data_ptr = lambda at=b.device(1).data_ptr(): at + 64  # of another layer
        refused(dev, hip.RstrError, "overlap the bounds", lambda: run(blocks=x))
        q = Dev((5, 4, 128))
        refused(dev, hip.RstrError, "overlap the queries", lambda: run(q=q, blocks=inside(ints((5, 2, 3)), q, 4 * (5 * 4 * 128 - 1))))
        n = dev.fake_launches()
        up(rows=0)
        run(q=Dev((0, 4, 128)), blocks=ints((0, 2, 3)))
        run(ro=ints(1), ln=ints(0), pt=ints((0, 7)))
        assert dev.fake_launches() == n


def test_the_callers_device_comes_back(dev):
    with hip.Session(1) as s:
        p = pool(s)
        dev.fake_device(0)
        row = Dev((1, 2, 128), device=1)
        p.rope_append(0, row, row, ints(1, device=1))
        b = hip.BlockBounds(p)
        b.close()
        assert dev.fake_device(-1) == 0


def test_arrays_without_a_length(dev):
    """data_ptr(), shape, stride(), dtype and device are enough."""
    with hip.Session(0) as s:
        p = pool(s, 1)
        keep = [Dev((2, 2, 128)), Dev((2, 2, 128)), ints(2), ints(2), Dev((64,), "float64"), Dev((2, 4, 128)), Dev((2, 4, 128)), ints(3), ints((2, 5)),
                ints(2), ints((2, 2, 3))]
        k, v, slots, pos, fr, q, out, offs, table, lens, blocks = [Bare(x) for x in keep]
        n = dev.fake_launches()
        p.rope_append(0, k, v, slots, pos, fr, q=q)
        b = hip.BlockBounds(p)
        b.update(0, offs, table, lens, 2)
        hip.BlockSelect(b, 4, 2, 2, 5).run(0, q, offs, table, lens, blocks)
        hip.PagedAttention(p, 4, 2, 2).run(0, q, offs, table, lens, out, blocks=blocks)
        assert dev.fake_launches() == n + 4
