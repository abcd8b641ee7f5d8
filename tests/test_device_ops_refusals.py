"""What the operators on device arrays refuse, and that they do so before any
device work: the C entries and their Python twin over a device that only counts
launches (tests/native/fake_device.cpp), no GPU needed."""
import ctypes as C
import os
import shutil
import subprocess

import numpy as np
import pytest

from rstr import hip

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "pretrained-rstr_amd", "csrc")
NEW = [n for n in hip.EXPORTS if n.startswith(("rstr_kv4", "rstr_verify", "rstr_step_maps"))]
BASE = ["rstr_session_open", "rstr_session_close", "rstr_last_error", "rstr_open_error"]

pytestmark = pytest.mark.skipif(shutil.which("hipcc") is None, reason="no hipcc")


@pytest.fixture(scope="module")
def fake_lib(tmp_path_factory):
    tmp = tmp_path_factory.mktemp("fake")
    so = str(tmp / "librstr_fake.so")
    objects = []
    for src in (os.path.join(CSRC, "device_ops.cpp"), os.path.join(HERE, "native", "fake_device.cpp")):
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


class Dev:
    """An array that says it lives on a GPU."""

    def __init__(self, shape, dtype="float32", device=0, strides=None, shift=0):
        n = {"float16": "f2", "bfloat16": "u2"}.get(dtype, dtype)
        self._keep = np.zeros(int(np.prod(shape)) * 4 + 64, n)
        self.shape, self.dtype, self.device, self._shift = tuple(shape), dtype, device, shift
        self._st = strides or tuple(int(np.prod(self.shape[i + 1:])) for i in range(len(shape)))

    def __len__(self):
        return self.shape[0]

    def data_ptr(self):
        return self._keep.ctypes.data + self._shift

    def stride(self):
        return self._st


def ints(n, **kw):
    return Dev(n if isinstance(n, tuple) else (n,), "int32", **kw)


def refused(dev, exc, match, call):
    before = dev.fake_launches()
    with pytest.raises(exc, match=match):
        call()
    assert dev.fake_launches() == before


def test_cache_open(dev):
    blocks = dev.fake_blocks()
    with hip.Session(0) as s:
        for args, match in (((0, 2, 128, 16, 4), "extents"), ((1, 0, 128, 16, 4), "extents"), ((1, 2, 128, 0, 4), "extents"),
                            ((1, 2, 128, 16, 0), "extents"), ((1, 2, 96, 16, 4), "head dim"), ((1, 2, 128, 24, 4), "multiple of 16"),
                            ((1, 2, 128, 1 << 16, 1 << 15), "31 bits"), ((1, 2, 64, 1 << 24, 1), "2 GB")):
            with pytest.raises(hip.RstrError, match=match) as e:
                hip.Kv4Pool(s, *args)
            assert e.value.code == -1
        dev.fake_fail_alloc(1)
        try:
            with pytest.raises(hip.RstrError) as e:
                hip.Kv4Pool(s, 1, 2, 128, 16, 4)
            assert e.value.code == -3
            with pytest.raises(hip.RstrError) as e:
                hip.Verifier(s, 1, 1, 10)
            assert e.value.code == -3
        finally:
            dev.fake_fail_alloc(0)
        p = hip.Kv4Pool(s, 3, 2, 128, 16, 4)
        assert p.nbytes == 3 * 2 * 4 * 16 * 144
        plan = hip.Kv4Attention(p, 4, 2, 5)
        with pytest.raises(hip.RstrError, match="open attention plans") as e:
            p.close()
        assert e.value.code == -4
        plan.close()
        plan.close()
        p.close()
        for n_q in (0, 3):
            q = hip.Kv4Pool(s, 1, 2, 64, 16, 4)
            with pytest.raises(hip.RstrError, match="query heads"):
                hip.Kv4Attention(q, n_q, 2, 5)
            with pytest.raises(hip.RstrError, match="too many rows"):
                hip.Kv4Attention(q, 64, 1, 1 << 26)
        with pytest.raises(hip.RstrError, match="vocabulary"):
            hip.Verifier(s, 1, 1, (1 << 24) + 1)
    assert dev.fake_blocks() == blocks


def test_null_handles(dev):
    z = [0] * 20
    for name in NEW:
        f = getattr(dev, name)
        if name.endswith(("_close",)):
            assert f(None) == 0
        elif name == "rstr_kv4_bytes":
            assert f(None) == -1
        else:
            args = [None if t in (C.c_void_p,) or isinstance(t, type(C.POINTER(C.c_void_p))) else z[0] for t in f.argtypes]
            assert f(*args) == -1, name


def test_rows(dev):
    with hip.Session(0) as s:
        p = hip.Kv4Pool(s, 2, 2, 128, 16, 4)
        k, v, sl = Dev((3, 2, 128)), Dev((3, 2, 128)), ints(3)
        for op in (lambda **a: p.append(a.get("layer", 0), a.get("k", k), a.get("v", v), a.get("slots", sl), stream=7),
                   lambda **a: p.read(a.get("layer", 0), a.get("slots", sl), a.get("k", k), a.get("v", v), stream=7)):
            op()
            assert dev.fake_stream() == 7
            refused(dev, hip.RstrError, "layer", lambda: op(layer=2))
            refused(dev, hip.RstrError, "layer", lambda: op(layer=-1))
            refused(dev, ValueError, "shape", lambda: op(k=Dev((3, 3, 128))))
            refused(dev, ValueError, "shape", lambda: op(k=Dev((4, 2, 128))))
            refused(dev, ValueError, "shape", lambda: op(v=Dev((3, 2, 64))))
            refused(dev, ValueError, "same element type", lambda: op(v=Dev((3, 2, 128), "float16")))
            refused(dev, ValueError, "float32, float16 or bfloat16", lambda: op(k=Dev((3, 2, 128), "float64")))
            refused(dev, ValueError, "last dimension", lambda: op(k=Dev((3, 2, 128), strides=(512, 256, 2))))
            refused(dev, ValueError, "session's GPU", lambda: op(k=Dev((3, 2, 128), device=1)))
            refused(dev, ValueError, "int32", lambda: op(slots=Dev((3,), "int64")))
            refused(dev, ValueError, "contiguous", lambda: op(slots=ints(3, strides=(2,))))
            refused(dev, hip.RstrError, "aligned", lambda: op(k=Dev((3, 2, 128), shift=2)))
            refused(dev, hip.RstrError, "aligned", lambda: op(slots=ints(3, shift=1)))
            refused(dev, hip.RstrError, "strides", lambda: op(k=Dev((3, 2, 128), strides=(-256, 128, 1))))
            n = dev.fake_launches()
            op(k=Dev((0, 2, 128)), v=Dev((0, 2, 128)), slots=ints(0))
            assert dev.fake_launches() == n  # nothing to do, nothing queued
        refused(dev, hip.RstrError, "share elements", lambda: p.read(0, sl, Dev((3, 2, 128), strides=(64, 128, 1)), v))
        refused(dev, hip.RstrError, "share elements", lambda: p.read(0, sl, k, Dev((3, 2, 128), strides=(0, 128, 1))))
        p.read(0, sl, Dev((3, 2, 128), strides=(128, 384, 1)), v, stream=0)  # heads outside, rows inside: apart
        p.append(0, Dev((3, 2, 128), strides=(0, 128, 1)), v, sl)            # a broadcast row may be read


def test_attention(dev):
    with hip.Session(0) as s:
        p = hip.Kv4Pool(s, 2, 2, 128, 16, 4)
        plan = hip.Kv4Attention(p, 4, 2, 5)

        def run(**kw):
            a = {**dict(layer=0, q=Dev((5, 4, 128)), ro=ints(3), pt=ints((2, 7)), ln=ints(2), out=Dev((5, 4, 128))), **kw}
            plan.run(*[a.pop(n) for n in ("layer", "q", "ro", "pt", "ln", "out")], **a)

        run()
        run(stream=hip.SESSION_STREAM)
        assert dev.fake_stream() == 0x5e55
        run(max_rows=3, window=4, scale=0.5)
        for match, kw in (("layer", dict(layer=2)), ("window", dict(window=-1)), ("scale", dict(scale=float("nan"))),
                          ("rows per sequence", dict(max_rows=0)), ("rows per sequence", dict(max_rows=6)),
                          ("batch exceeds", dict(ro=ints(4), ln=ints(3), pt=ints((3, 7)))),
                          ("rows exceed", dict(q=Dev((6, 4, 128)), out=Dev((6, 4, 128)))),
                          ("width", dict(pt=ints((2, 0)))), ("share elements", dict(out=Dev((5, 4, 128), strides=(128, 128, 1)))),
                          ("aligned", dict(q=Dev((5, 4, 128), "float16", shift=1), out=Dev((5, 4, 128), "float16")))):
            refused(dev, hip.RstrError, match, lambda: run(**kw))
        for match, kw in (("shape", dict(q=Dev((5, 3, 128)))), ("shape", dict(out=Dev((4, 4, 128)))),
                          ("same element type", dict(out=Dev((5, 4, 128), "float16"))), ("shape", dict(ro=ints(4))),
                          ("shape", dict(pt=ints((3, 7)))), ("int32", dict(ln=Dev((2,), "float32"))),
                          ("contiguous", dict(pt=ints((2, 7), strides=(14, 1)))), ("session's GPU", dict(pt=ints((2, 7), device=3)))):
            refused(dev, ValueError, match, lambda: run(**kw))
        x = Dev((5, 4, 128))
        refused(dev, hip.RstrError, "overlaps the queries", lambda: run(q=x, out=x))
        n = dev.fake_launches()
        run(q=Dev((0, 4, 128)), out=Dev((0, 4, 128)))
        run(ro=ints(1), ln=ints(0), pt=ints((0, 7)))
        assert dev.fake_launches() == n


def test_the_callers_device_comes_back(dev):
    with hip.Session(1) as s:
        p = hip.Kv4Pool(s, 1, 2, 128, 16, 4)
        dev.fake_device(0)
        p.append(0, Dev((1, 2, 128), device=1), Dev((1, 2, 128), device=1), ints(1, device=1))
        assert dev.fake_device(-1) == 0
        p.close()
        assert dev.fake_device(-1) == 0


def test_step_maps(dev):
    with hip.Session(0) as s:
        base = dict(lengths=ints(2), counts=ints(2), free_pages=ints(6), page_table=ints((2, 5)), new_lengths=ints(2),
                    row_offsets=ints(3), positions=ints(4), slots=ints(4), taken=ints(1))

        def run(page=16, **kw):
            s.step_maps(page, **{**base, **kw})

        run()
        run(starts=ints(2))
        run(free_pages=ints(0), positions=ints(0), slots=ints(0))
        refused(dev, hip.RstrError, "extents", lambda: run(page=0))
        refused(dev, hip.RstrError, "extents", lambda: run(page_table=ints((2, 0))))
        refused(dev, hip.RstrError, "overlap", lambda: run(new_lengths=base["lengths"]))
        refused(dev, hip.RstrError, "overlap", lambda: run(positions=base["slots"]))
        refused(dev, hip.RstrError, "overlap", lambda: run(starts=base["new_lengths"]))
        refused(dev, hip.RstrError, "aligned", lambda: run(starts=ints(2, shift=2)))
        n = 8193
        refused(dev, hip.RstrError, "batch", lambda: run(lengths=ints(n), counts=ints(n), page_table=ints((n, 5)), new_lengths=ints(n),
                                                        row_offsets=ints(n + 1)))
        refused(dev, hip.RstrError, "batch", lambda: run(lengths=ints(0), counts=ints(0), page_table=ints((0, 5)), new_lengths=ints(0),
                                                        row_offsets=ints(1)))
        for kw in (dict(counts=ints(3)), dict(page_table=ints((3, 5))), dict(row_offsets=ints(2)), dict(positions=ints(3)),
                   dict(taken=ints(2)), dict(starts=ints(1))):
            refused(dev, ValueError, "shape", lambda: run(**kw))


def test_verify(dev):
    with hip.Session(0) as s:
        v = hip.Verifier(s, 2, 5, 100)
        base = dict(logits=Dev((5, 100)), row_offsets=ints(3), drafts=ints(5), temperature=Dev((2,)), u_accept=Dev((5,)),
                    u_sample=Dev((2,)), accepted=ints(2), tokens=ints(5))

        def run(**kw):
            v.run(**{**base, **kw})

        run()
        run(draft_probs=Dev((5, 100)), logits=Dev((5, 100), "bfloat16", strides=(112, 1)))
        n = dev.fake_launches()
        run(row_offsets=ints(1), temperature=Dev((0,)), u_sample=Dev((0,)), accepted=ints(0))  # no sequences
        assert dev.fake_launches() == n
        refused(dev, hip.RstrError, "batch exceeds", lambda: run(row_offsets=ints(4), temperature=Dev((3,)), u_sample=Dev((3,)), accepted=ints(3)))
        refused(dev, hip.RstrError, "rows exceed", lambda: run(logits=Dev((6, 100)), drafts=ints(6), u_accept=Dev((6,)), tokens=ints(6)))
        refused(dev, hip.RstrError, "overlap", lambda: run(tokens=base["drafts"]))
        for name in ("tokens", "accepted"):   # inside the logits' last row
            x = Dev((5, 100))
            inside = ints(5 if name == "tokens" else 2)
            inside._keep, inside._shift = x._keep, 4 * 499
            refused(dev, hip.RstrError, "overlap", lambda: run(logits=x, **{name: inside}))
        refused(dev, hip.RstrError, "aligned", lambda: run(logits=Dev((5, 100), shift=2)))
        for match, kw in (("shape", dict(logits=Dev((5, 99)))), ("last dimension", dict(logits=Dev((5, 100), strides=(200, 2)))),
                          ("must be float32", dict(draft_probs=Dev((5, 100), "float16"))), ("float32", dict(temperature=Dev((2,), "float16"))),
                          ("shape", dict(u_sample=Dev((5,)))), ("int32", dict(drafts=Dev((5,), "int64"))),
                          ("session's GPU", dict(logits=Dev((5, 100), device=1)))):
            refused(dev, ValueError, match, lambda: run(**kw))


def inside(x, other, at):
    """The array x over the memory of another, from byte `at` on."""
    x._keep, x._shift = other._keep, at
    return x


def test_reads_into_shared_memory(dev):
    with hip.Session(0) as s:
        p = hip.Kv4Pool(s, 1, 2, 128, 16, 4)
        sl = ints(3)
        one = Dev((3, 2, 2, 128))
        read = lambda at, strides: p.read(0, sl, inside(Dev((3, 2, 128), strides=strides), one, 0), inside(Dev((3, 2, 128), strides=strides), one, 4 * at))  # noqa: E731
        read(256, (512, 128, 1))     # [rows][k, v][heads][head_dim]
        read(128, (512, 256, 1))     # [rows][heads][k, v][head_dim]
        read(384, (128, 768, 1))     # [heads][k, v][rows][head_dim]
        read(128, (256, 768, 1))     # [heads][rows][k, v][head_dim]
        read(768, (256, 128, 1))     # one behind the other
        read(384 * 2, (128, 384, 1))
        for at, strides in ((0, (256, 128, 1)), (128, (512, 128, 1)), (255, (512, 128, 1)), (127, (512, 256, 1)), (256, (256, 128, 1)),
                            (257, (512, 128, 1)), (383, (128, 768, 1)), (64, (512, 256, 1)), (640, (256, 128, 1))):
            refused(dev, hip.RstrError, "share elements", lambda: read(at, strides))
        k, v = Dev((3, 2, 128)), Dev((3, 2, 128))
        refused(dev, hip.RstrError, "overlap the slots", lambda: p.read(0, inside(ints(3), k, 4 * 767), k, v))
        refused(dev, hip.RstrError, "overlap the slots", lambda: p.read(0, inside(ints(3), v, 0), k, v))
        p.read(0, inside(ints(3), v, 4 * 768), k, v)


def test_outputs_inside_tables_and_probabilities(dev):
    with hip.Session(0) as s:
        p = hip.Kv4Pool(s, 2, 2, 128, 16, 4)
        plan = hip.Kv4Attention(p, 4, 2, 5)
        out = Dev((5, 4, 128))
        for which, a in enumerate((ints(3), ints((2, 7)), ints(2))):
            tables = [ints(3), ints((2, 7)), ints(2)]
            tables[which] = inside(a, out, 4 * (5 * 4 * 128 - 1))
            refused(dev, hip.RstrError, "overlaps the sequences' tables", lambda: plan.run(0, Dev((5, 4, 128)), *tables, out))
            tables[which] = inside(a, out, 4 * 5 * 4 * 128)
            plan.run(0, Dev((5, 4, 128)), *tables, out)
        v = hip.Verifier(s, 2, 5, 100)
        base = dict(logits=Dev((5, 100)), row_offsets=ints(3), drafts=ints(5), temperature=Dev((2,)), u_accept=Dev((5,)), u_sample=Dev((2,)),
                    accepted=ints(2), tokens=ints(5))
        for name, n in (("tokens", 5), ("accepted", 2)):
            probs = Dev((5, 100))
            refused(dev, hip.RstrError, "overlap", lambda: v.run(**{**base, name: inside(ints(n), probs, 4 * 499)}, draft_probs=probs))
            v.run(**{**base, name: inside(ints(n), probs, 4 * 500)}, draft_probs=probs)


def test_plans_past_a_grid(dev):
    """Rows or sequences of which a launch cannot have a workgroup each."""
    blocks = dev.fake_blocks()
    with hip.Session(0) as s:
        p = hip.Kv4Pool(s, 1, 8, 64, 16, 4)
        for n_q, batch, rows in ((8, 1 << 22, 1 << 22), (32, 1, (1 << 26) - 1024), (8, 1, 1 << 25)):
            with pytest.raises(hip.RstrError, match="too many rows"):
                hip.Kv4Attention(p, n_q, batch, rows)
        hip.Kv4Attention(p, 8, 1 << 20, 1 << 20).close()
        hip.Kv4Attention(p, 32, 1 << 20, 1 << 17).close()
        for batch, rows in ((1, 1 << 24), (1 << 24, 1), (1, 2 ** 31 - 1)):
            with pytest.raises(hip.RstrError, match="too many rows"):
                hip.Verifier(s, batch, rows, 2)
        hip.Verifier(s, 1 << 23, 1 << 23, 2).close()
        p.close()
    assert dev.fake_blocks() == blocks


class Bare:
    """An array with nothing but what the operators ask of one."""

    def __init__(self, x):
        self.data_ptr, self.shape, self.stride, self.dtype, self.device = x.data_ptr, x.shape, x.stride, x.dtype, x.device


def test_arrays_without_a_length(dev):
    """data_ptr(), shape, stride(), dtype and device are enough."""
    with hip.Session(0) as s:
        keep = [Dev((2, 2, 128)), Dev((2, 2, 128)), ints(2), Dev((2, 4, 128)), Dev((2, 4, 128)), ints(3), ints((2, 5)), ints(2), ints(2), ints(2), ints(1),
                ints(6), Dev((2, 100)), Dev((2,)), Dev((2,)), Dev((2,)), ints(2), ints(2)]
        k, v, slots, q, out, offs, table, lens, more, pos, one, free, logits, T, ua, us, acc, tok = [Bare(x) for x in keep]
        n = dev.fake_launches()
        p = hip.Kv4Pool(s, 1, 2, 128, 16, 4)
        p.append(0, k, v, slots)
        p.read(0, slots, k, v)
        hip.Kv4Attention(p, 4, 2, 2).run(0, q, offs, table, lens, out)
        s.step_maps(16, lens, more, free, table, acc, offs, pos, slots, one)
        hip.Verifier(s, 2, 2, 100).run(logits, offs, slots, T, ua, us, acc, tok)
        view = hip.DeviceView(keep[12].data_ptr(), (2, 100), "float32", 0, None)
        hip.Verifier(s, 2, 2, 100).run(view, offs, slots, T, ua, us, acc, tok)
        assert dev.fake_launches() == n + 6
