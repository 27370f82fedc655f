"""The batched-serving calls without a GPU: their refusals, through the C ABI, launch nothing; the cache
addressing and the division of the work run on the host from the header that the kernels include."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

from g4b import _lib as L

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(REPO, "gemma4-12b-snapdragonx2elite_b200", "csrc")


@pytest.fixture(scope="module")
def buf():
    raw = C.create_string_buffer(4096 + 16)
    yield (C.addressof(raw) + 15) & ~15
    del raw


SIZES = dict(T=4, B=2, nH=16, nkv=8, hd=256, page_size=64, table_pages=4, prefix_pages=2, window=0)


def _sizes(**kw):
    return tuple(dict(SIZES, **kw).values())


def _plan(p, plan_bytes=1 << 40, prefix_len=True, plan=None, **kw):
    return L.load().g4b_paged_plan(p, p, p if prefix_len else None, *_sizes(**kw), p if plan is None else plan,
                                   plan_bytes, None)


def _append(p, dtype=1, row_stride=8192, n_pos=384, num_pages=8, q_stride=4096, koff=4096, voff=6144, qkv=None, **kw):
    s = _sizes(**kw)
    return L.load().g4b_paged_append(p if qkv is None else qkv, dtype, row_stride, p, p, p, p, n_pos, p, p, num_pages, p,
                                     p, q_stride, *s[:5], koff, voff, *s[5:], p, None)


def _attn(p, q_stride=4096, num_pages=8, prefix_table=True, out_dtype=1, out_stride=4096, scale=1.0, ws=None,
          ws_bytes=1 << 40, q=None, **kw):
    return L.load().g4b_paged_attn(p if q is None else q, q_stride, p, p, num_pages, p, p if prefix_table else None, p,
                                   out_dtype, out_stride, scale, *_sizes(**kw), p, p if ws is None else ws, ws_bytes,
                                   None)


BAD_SIZES = [dict(T=0), dict(B=0), dict(B=4097), dict(nkv=0), dict(nH=12), dict(nH=4), dict(hd=64), dict(hd=192),
             dict(page_size=8), dict(page_size=48), dict(page_size=2048), dict(table_pages=0), dict(prefix_pages=-1),
             dict(window=-1), dict(table_pages=1 << 25), dict(T=1 << 26)]


@pytest.mark.parametrize("bad", BAD_SIZES, ids=str)
def test_sizes_are_refused(buf, bad):
    for call in (_plan, _append, _attn):
        assert call(buf, **bad) == L.G4B_E_SHAPE, (call, bad)
    lib = L.load()
    assert lib.g4b_paged_plan_bytes(*_sizes(**bad)) == 0 and L.last_error()
    assert lib.g4b_paged_workspace_bytes(*_sizes(**bad)) == 0 and L.last_error()


def test_sizes_of_plan_and_workspace():
    lib = L.load()
    small, big = (lib.g4b_paged_plan_bytes(*_sizes(T=t)) for t in (4, 4096))
    assert 0 < small < big
    # without a prefix the workspace does not grow with the tokens
    a, b = (lib.g4b_paged_workspace_bytes(*_sizes(T=t, prefix_pages=0)) for t in (4, 4096))
    assert 0 < a == b < lib.g4b_paged_workspace_bytes(*_sizes(T=4096))


def test_plan_refusals(buf):
    assert L.load().g4b_paged_plan(None, buf, buf, *_sizes(), buf, 1 << 40, None) == L.G4B_E_ARG
    assert _plan(buf, prefix_len=False) == L.G4B_E_ARG
    assert _plan(buf, plan_bytes=16) == L.G4B_E_WORKSPACE
    assert _plan(buf, plan=buf + 4) == L.G4B_E_ALIGN


def test_append_refusals(buf):
    assert _append(buf, dtype=3) == L.G4B_E_ARG
    for bad in (dict(num_pages=0), dict(num_pages=1 << 23), dict(n_pos=383), dict(koff=4097), dict(voff=-8),
                dict(row_stride=8188), dict(row_stride=8184), dict(q_stride=4088), dict(voff=6152)):
        assert _append(buf, **bad) == L.G4B_E_SHAPE, bad
    assert _append(buf, qkv=buf + 8) == L.G4B_E_ALIGN
    assert "16-byte" in L.last_error()


def test_attention_refusals(buf):
    assert _attn(buf, out_dtype=2) == L.G4B_E_ARG
    assert _attn(buf, prefix_table=False) == L.G4B_E_ARG
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        assert _attn(buf, scale=scale) == L.G4B_E_ARG
    for bad in (dict(num_pages=0), dict(num_pages=1 << 23), dict(q_stride=4088), dict(out_stride=4100)):
        assert _attn(buf, **bad) == L.G4B_E_SHAPE, bad
    assert _attn(buf, q=buf + 2) == L.G4B_E_ALIGN
    assert _attn(buf, ws_bytes=64) == L.G4B_E_WORKSPACE
    assert _attn(buf, ws=buf + 4) == L.G4B_E_WORKSPACE


def test_normadd_i8_refusals(buf):
    f = L.load().g4b_rows_normadd_i8
    p = buf
    assert f(p, 1, p, None, p, 1.0, p, p, p, 4, 256, None) == L.G4B_E_ARG
    assert f(None, 1, p, p, p, 1.0, p, p, p, 4, 256, None) == L.G4B_E_ARG           # w_post without x
    assert f(p, 2, p, p, p, 1.0, p, p, p, 4, 256, None) == L.G4B_E_ARG
    assert f(p, 1, p, p, p + 64, 1.0, p, p, p, 4, 256, None) == L.G4B_E_ARG         # h_out overlaps h
    for m, d in ((0, 256), (4, 8), (4, 24), (-1, 16)):
        assert f(p, 1, p, p, p, 1.0, p, p, p, m, d, None) == L.G4B_E_SHAPE
    q = (p + 31) & ~31
    for i in (0, 2, 3, 4, 6, 7, 8):             # x, w_post, h, h_out, w, A8, sa
        args = [q, 1, q, q, q, 1.0, q, q, q, 4, 256, None]
        args[i] += 2 if i == 8 else 8 if i == 7 else 16
        if i in (3, 4):
            args[3] = args[4] = q + 16
        assert f(*args) == L.G4B_E_ALIGN


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    """The header's functions, compiled for the host."""
    d = tmp_path_factory.mktemp("pages")
    src, so = d / "pages.cpp", d / "pages.so"
    src.write_text('#include "g4b_pages.h"\nextern "C" {\n'
                   "int row(int p, int n, int k, int s, int h, int key) "
                   "{ return g4b::pg::cache_row(p, n, k, __builtin_ctz(s), h, key); }\n"
                   "void span(long long g, int n, long long u, int* o) "
                   "{ auto s = g4b::pg::span_of(g, n, u); o[0] = s.c0; o[1] = s.c1; }\n}\n")
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-I", CSRC, str(src), "-o", str(so)], check=True)
    lib = C.CDLL(str(so))
    lib.span.argtypes = [C.c_longlong, C.c_int, C.c_longlong, C.c_void_p]
    return lib


def test_rows_of_pages_and_of_pages_that_are_not_there(host):
    pages, nkv, ps = 7, 3, 32
    for page in range(pages):
        for head in range(nkv):
            for key in (0, 1, ps - 1, ps, 5 * ps + 3):
                r = host.row(page, pages, nkv, ps, head, key)
                assert r == np.ravel_multi_index((page, head, key % ps), (pages, nkv, ps))
    for page in (-1, -2**31, pages, 2**31 - 1):
        assert host.row(page, pages, nkv, ps, 0, 0) == -1
    # the largest cache a call takes: the row still fits 32 bits
    assert host.row(2**20 - 2, 2**20 - 1, 2, 1024, 1, 1023) == (2**20 - 1) * 2 * 1024 - 1


def test_spans_cover_the_line_of_work(host):
    rng = np.random.default_rng(0)
    for _ in range(50):
        n = rng.integers(0, 40, rng.integers(1, 30))
        total = int(n.sum())
        if total == 0:
            continue
        ctas = int(rng.integers(1, 20))
        u = max(1, -(-total // ctas))
        off, owner = 0, np.repeat(np.arange(-(-total // u)), u)[:total]
        for k in n:
            if k:
                o = np.zeros(2, np.int32)
                host.span(off, int(k), u, o.ctypes.data)
                assert o[0] == owner[off] and o[1] == owner[off + k - 1] and o[1] < ctas
            off += int(k)


@pytest.fixture(scope="module")
def overlap(tmp_path_factory):
    d = tmp_path_factory.mktemp("overlap")
    src, so = d / "overlap.cpp", d / "overlap.so"
    src.write_text('#include "g4b_overlap.h"\nextern "C" int overlap(long long p, long long n, long long s, long long w, '
                   "long long q, long long m, long long t, long long v) { return g4b::rows_overlap("
                   "{reinterpret_cast<void*>(p), n, s, w}, {reinterpret_cast<void*>(q), m, t, v}); }\n")
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-I", CSRC, str(src), "-o", str(so)], check=True)
    lib = C.CDLL(str(so))
    lib.overlap.argtypes = [C.c_longlong] * 8
    return lib.overlap


def test_overlap_of_rows(overlap):
    """Against the sets of bytes, for buffers of one stride; differing strides may only err towards an overlap."""
    rng = np.random.default_rng(1)
    seen = set()
    for _ in range(4000):
        n, m, s, t = (int(x) for x in rng.integers(1, 6, 4))
        s, t = 8 * s, 8 * (s if rng.random() < 0.7 else t)
        w, v = int(rng.integers(1, s + 1)), int(rng.integers(1, t + 1))
        p, q = (int(x) for x in 100 + rng.integers(0, 120, 2))
        a = {p + i * s + j for i in range(n) for j in range(w)}
        b = {q + i * t + j for i in range(m) for j in range(v)}
        got = overlap(p, n, s, w, q, m, t, v)
        assert got == bool(a & b) if s == t else got >= bool(a & b), (p, n, s, w, q, m, t, v)
        seen.add((s == t, got))
    assert len(seen) == 4
    assert not overlap(0, 1, 8, 8, 0, 1, 8, 8)               # a buffer that is not given


FAR = 1 << 40      # addresses that nothing reads: a call that is refused launches nothing


def test_buffers_that_overlap_are_refused():
    lib, s = L.load(), _sizes(prefix_pages=0)
    q, kc, vc, out, ws = FAR, FAR + (1 << 32), FAR + (2 << 32), FAR + (3 << 32), FAR + (4 << 32)

    def attn(q=q, kc=kc, vc=vc, out=out, out_dtype=1, stride=4096):
        return lib.g4b_paged_attn(q, stride, kc, vc, 8, FAR, None, out, out_dtype, stride, 1.0, *s, FAR, ws, 1 << 40, None)

    for bad in (dict(out=q), dict(out=q + 2 * 4096), dict(out=kc + 4096), dict(out=vc - 64), dict(out=q - 64),
                dict(out=q + 4096, stride=8192), dict(out=q + 2 * 4096, stride=8192, out_dtype=0)):
        assert attn(**bad) == L.G4B_E_ARG, bad
        assert "overlap" in L.last_error()

    def append(qkv=q, kc=kc, vc=vc, q_out=out):
        return lib.g4b_paged_append(qkv, 1, 8192, ws, ws, ws, ws, 384, kc, vc, 8, ws, q_out, 4096, *s[:5], 4096, 6144,
                                    *s[5:], ws, None)

    for bad in (dict(vc=kc), dict(vc=kc + 64), dict(q_out=q), dict(q_out=kc), dict(qkv=vc + 128)):
        assert append(**bad) == L.G4B_E_ARG, bad
        assert "overlap" in L.last_error()


def test_normadd_i8_refuses_buffers_that_overlap():
    x, h, w, h_out, a8, sa = (FAR + (i << 32) for i in range(6))
    M, D = 4, 256
    good = dict(x=x, w_post=w + 4096, h=h, h_out=h_out, w=w, a8=a8, sa=sa)
    for bad in (dict(x=h_out), dict(x=h, h_out=h), dict(w=h_out + 64), dict(w_post=h_out), dict(a8=h), dict(a8=x + 32),
                dict(sa=a8 + 64), dict(sa=w), dict(a8=h_out + 4 * M * D - 32), dict(h_out=h + 32)):
        p = dict(good, **bad)
        assert L.load().g4b_rows_normadd_i8(p["x"], 1, p["w_post"], p["h"], p["h_out"], 1.0, p["w"], p["a8"], p["sa"], M, D,
                                            None) == L.G4B_E_ARG, bad
        assert "overlap" in L.last_error()


def test_a_stream_of_another_device_is_refused():
    from types import SimpleNamespace

    from g4b import ops
    with pytest.raises(ValueError, match="cuda:1"):
        ops._on(0, SimpleNamespace(device_index=1))


# sizes whose hash to a word was the same for 148 SMs, as in PlanKey: T, B, nH, nkv, hd, page_size, tables, window, CTAs
TWINS = ((67, 67, 16, 8, 256, 64, 29, 16, 1024, 296, 148), (128, 128, 16, 8, 256, 64, 12, 32, 1024, 296, 148))


def test_a_plan_is_taken_for_its_own_sizes_only(tmp_path):
    src, so = tmp_path / "key.cpp", tmp_path / "key.so"
    src.write_text('#include "g4b_pages.h"\nextern "C" int same(const int* a, const int* b) {\n'
                   "g4b::pg::PlanKey x{}, y{};\n"
                   "for (int i = 0; i < 12; i++) { x.v[i] = a[i]; y.v[i] = b[i]; }\n"
                   "return g4b::pg::same_plan(x, y); }\nextern \"C\" int magic() { return g4b::pg::kPlanMagic; }\n")
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-I", CSRC, str(src), "-o", str(so)], check=True)
    lib = C.CDLL(str(so))
    key = lambda *v: (C.c_int * 12)(*v)  # noqa: E731
    a, b = (key(lib.magic(), *t) for t in TWINS)
    assert lib.magic() != 0 and lib.same(a, a) and lib.same(b, b) and not lib.same(a, b)
    for i in range(12):                      # no field may differ, by however little
        for bit in (0, 1, 8, 31):
            c = key(*a)
            c[i] = np.int32(np.uint32(c[i]) ^ np.uint32(1 << bit))
            assert not lib.same(a, c) and not lib.same(c, a)
    assert not lib.same(key(*[0] * 12), a)


def test_rows_too_long_to_count_are_refused():
    x, h, w, h_out, a8, sa = (FAR + (i << 36) for i in range(6))
    f = L.load().g4b_rows_normadd_i8
    for d in ((1 << 30) + 16, 2**31 - 16):
        assert f(x, 1, None, h, h_out, 1.0, w, a8, sa, 1, d, None) == L.G4B_E_SHAPE and "2^30" in L.last_error()
    assert f(x, 1, None, h, h_out, 1.0, w, h + 32, sa, 1, 1 << 30, None) == L.G4B_E_ARG      # that size is looked at further


def test_a_plan_on_the_host_is_refused():
    from g4b.paged import PagedPlan
    for device in ("cpu", "meta"):
        with pytest.raises(ValueError, match=device):
            PagedPlan(1, 1, 16, 8, 256, 64, 1, device=device)
