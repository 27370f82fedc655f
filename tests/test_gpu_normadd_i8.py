"""g4b_rows_normadd_i8 against its definition in 64 bits, against the three calls that it stands for, and in a batched
layer's run of append, attention, W8A8 GEMMs and norm.

Tolerances count roundings of 2^-24: h' makes under 16 (its norm factor among them) on terms no larger than
(|h| + |x^ w_post|) scl; sa another 16; a code lies within half a step of y / sa, whose own error is at most
|code| 2^-19."""
import numpy as np
import pytest
import torch

from g4b import _lib as L
from g4b import ops
from g4b.paged import PagedPlan

pytestmark = pytest.mark.gpu
DEV = "cuda"
F64 = torch.float64
ULP = 2.0 ** -20      # 16 roundings


def _definition(x, h, w, w_post, scl):
    x = None if x is None else x.to(F64)
    h = h.to(F64)
    add = torch.zeros_like(h)
    if x is not None:
        add = x if w_post is None else x * (x.pow(2).mean(-1, keepdim=True) + 1e-6).rsqrt() * w_post.to(F64)
    h1 = (h + add) * scl
    y = h1 * (h1.pow(2).mean(-1, keepdim=True) + 1e-6).rsqrt() * w.to(F64)
    return h1, (h.abs() + add.abs()) * abs(scl), y, torch.clamp(y.abs().amax(-1) / 127, min=1e-12)


def _check(x, h, w, w_post, scl, h1, a8, sa, what=""):
    """The inputs as they were before the call, and what it gave."""
    rh, mag, ry, rs = _definition(x, h, w, w_post, scl)
    if h1 is not None:
        assert ((h1.to(F64) - rh).abs() <= ULP * mag + 1e-38).all(), what
    # the second norm's input carries h1's error: relative to the row's largest where terms cancel
    slack = 2.0 ** -19 + (ULP * mag).amax(-1) / rh.abs().amax(-1).clamp(min=1e-30)
    slack = torch.where(rs <= 1e-12, torch.full_like(slack, 1.0), slack)
    assert ((sa.to(F64) - rs).abs() <= 4 * slack * rs + 1e-18).all(), what
    real = ry / rs[:, None]
    code_err = (a8.to(F64) - real).abs()
    assert (code_err <= 0.5 + 127 * 8 * slack[:, None]).all(), f"{what}: {code_err.max().item()}"


SHAPES = [(1, 3840), (37, 3840), (3, 16), (5, 80), (130, 512), (4, 4112), (7, 5120), (2, 8192), (9, 15360), (3, 16384),
          (2, 16400), (3, 40000), (700, 256)]


@pytest.mark.parametrize("M,D", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("post,scl", [(True, 1.0), (True, 0.75), (False, 1.25)])
def test_matches_the_definition(M, D, dtype, post, scl):
    g = torch.Generator(device=DEV).manual_seed(M + D)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    x, h, w = (r(M, D) * torch.exp(r(M, 1))).to(dtype), 3 * r(M, D), 1 + 0.1 * r(D)
    w_post = 1 + 0.1 * r(D) if post else None
    out = torch.empty_like(h)
    h0 = h.clone()
    a8, sa = ops.rows_normadd_i8(x, h, w, w_post=w_post, scl=scl, h_out=out)
    torch.cuda.synchronize()
    assert torch.equal(h, h0)
    _check(x, h, w, w_post, scl, out, a8, sa)
    # in place, into given buffers: the same bits
    b8, sb = torch.empty_like(a8), torch.empty_like(sa)
    ops.rows_normadd_i8(x, h, w, w_post=w_post, scl=scl, A8=b8, sa=sb)
    torch.cuda.synchronize()
    assert torch.equal(h, out) and torch.equal(a8, b8) and torch.equal(sa, sb)


@pytest.mark.parametrize("M,D", [(1, 3840), (6, 15360), (2, 40000)])
def test_without_x(M, D):
    h, w = torch.randn(M, D, device=DEV), 1 + 0.1 * torch.randn(D, device=DEV)
    h0 = h.clone()
    a8, sa = ops.rows_normadd_i8(None, h, w)
    assert torch.equal(h, h0)
    _check(None, h0, w, None, 1.0, None, a8, sa)
    a8, sa = ops.rows_normadd_i8(None, h, w, scl=0.5)
    _check(None, h0, w, None, 0.5, h, a8, sa)


def test_near_the_three_calls():
    """rows_normadd, rows_rmsnorm, cast_i8: the residual within roundings, codes at most a step apart and nearly all equal."""
    M, D = 64, 3840
    g = torch.Generator(device=DEV).manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    x, h, w, wp = r(M, D).half(), 3 * r(M, D), 1 + 0.1 * r(D), 1 + 0.1 * r(D)
    h2 = h.clone()
    a8, sa = ops.rows_normadd_i8(x, h, w, w_post=wp, scl=0.75)
    ops.rows_normadd(x, wp, h2, 0.75)
    b8, sb = ops.cast_i8(ops.rows_rmsnorm(h2, w))
    assert ((h - h2).abs() <= ULP * (3 * h2.abs() + 8)).all()
    assert ((sa - sb).abs() <= 2.0 ** -18 * sb).all()
    d = (a8.int() - b8.int()).abs()
    assert d.max() <= 1 and (d > 0).float().mean() < 1e-3


def test_rows_of_zeros_large_and_tiny_values():
    D = 256
    h = torch.zeros(5, D, device=DEV)
    h[1] = 1e18
    h[2] = 1e-20
    h[3, 7] = -1e15
    h[4] = torch.randn(D, device=DEV) * 1e-3
    w = torch.ones(D, device=DEV)
    a8, sa = ops.rows_normadd_i8(torch.zeros(5, D, device=DEV), h.clone(), w)
    assert (a8[0] == 0).all() and sa[0].item() == np.float32(1e-12)
    assert (a8[1] == 127).all() and (a8[3, 7] == -127) and (a8[3].abs().sum() == 127)
    assert (a8[2] == 127).all() and abs(sa[2].item() * 127 / 1e-17 - 1) < 1e-3 or sa[2].item() == np.float32(1e-12)
    _check(None, h[4:], w, None, 1.0, None, a8[4:], sa[4:])


def test_python_refusals():
    h, w, x = torch.zeros(4, 256, device=DEV), torch.ones(256, device=DEV), torch.zeros(4, 256, device=DEV)
    with pytest.raises(ValueError):
        ops.rows_normadd_i8(x[:3], h, w)
    with pytest.raises(ValueError):
        ops.rows_normadd_i8(x, h[:, ::2], w)
    with pytest.raises(ValueError):
        ops.rows_normadd_i8(x.to(torch.bfloat16), h, w)
    with pytest.raises(ValueError):
        ops.rows_normadd_i8(x, h.half(), w)
    with pytest.raises(ValueError):
        ops.rows_normadd_i8(x, h, w.cpu())
    with pytest.raises(L.G4BError):
        ops.rows_normadd_i8(None, h, w, w_post=w)
    with pytest.raises(L.G4BError):
        ops.rows_normadd_i8(torch.zeros(4, 24, device=DEV), torch.zeros(4, 24, device=DEV), torch.ones(24, device=DEV))


def test_on_another_stream_and_in_a_graph():
    g = torch.Generator(device=DEV).manual_seed(2)
    x, h = torch.randn(50, 3840, generator=g, device=DEV), torch.randn(50, 3840, generator=g, device=DEV)
    w = 1 + 0.1 * torch.randn(3840, generator=g, device=DEV)
    h0, out = h.clone(), torch.empty_like(h)
    a8, sa = ops.rows_normadd_i8(x, h, w, h_out=out)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    b8, sb = ops.rows_normadd_i8(x, h, w, h_out=out, stream=s)
    s.synchronize()
    assert torch.equal(a8, b8) and torch.equal(sa, sb)
    c8, sc, out2 = torch.zeros_like(a8), torch.zeros_like(sa), torch.zeros_like(out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.rows_normadd_i8(x, h, w, h_out=out2, A8=c8, sa=sc)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(a8, c8) and torch.equal(sa, sc) and torch.equal(out, out2) and torch.equal(h, h0)


def test_a_batched_layer():
    """append -> attend -> W8A8 o -> normadd_i8 -> W8A8 gate, a layer of a batched step behind a shared prefix, against
    the same steps in 64 bits from the same int8 weights.  Every stage is compared from the stage's own inputs."""
    from test_gpu_paged import Batch, _append_reference, _close16
    nH, nkv, hd, D, I = 16, 8, 256, 3840, 512
    new, total, prefix = [1, 1, 3, 20, 1], [150, 131, 400, 161, 300], 130
    bt = Batch(nH, nkv, hd, 64, new, total, prefix, seed=30, back=2).fill()
    g = torch.Generator(device=DEV).manual_seed(31)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    qkv = r(bt.T, (nH + 2 * nkv) * hd).half()
    qnw, knw = 0.3 + 0.02 * r(hd), 1 + 0.1 * r(hd)
    ang = torch.arange((bt.own_pages + bt.pre_pages) * 64, device=DEV, dtype=F64)[:, None] * \
        10000.0 ** (-torch.arange(0, hd, 2, device=DEV, dtype=F64) / hd).repeat(2)
    cos, sin = ang.cos().float(), ang.sin().float()
    h = r(bt.T, D)
    paw, pfw = 1 + 0.1 * r(D), 1 + 0.1 * r(D)

    def weight(N, K):
        w8 = torch.randint(-127, 128, (K, N), generator=g, device=DEV, dtype=torch.int8)
        return ops.DeviceWeight(N=N, K=K, nblk=K // 32, split=1, scale_fmt=L.SCALE_F16, inv=1.0, wp=None, scales=None,
                                scales16=None, w8=w8, sw8=(1e-4 + 1e-4 * torch.rand(N, generator=g, device=DEV)).half())

    wo, wg = weight(D, nH * hd), weight(I, D)
    plan = bt.plan()
    q = plan.append(qkv, qnw, knw, cos, sin, bt.kc, bt.vc, bt.table, nH * hd, (nH + nkv) * hd)
    o = plan.attend(q, bt.kc, bt.vc, bt.table, bt.prefix_table, out=torch.zeros(bt.T, nH * hd, dtype=torch.float16, device=DEV))
    a8, sa = ops.cast_i8(o)
    t = ops.gemm_w8a8(a8, sa, wo)
    h1 = torch.empty_like(h)
    n8, sn = ops.rows_normadd_i8(t, h, pfw, w_post=paw, scl=0.9, h_out=h1)
    y = ops.gemm_w8a8(n8, sn, wg, out_dtype=torch.float32) if "out_dtype" in ops.gemm_w8a8.__code__.co_varnames \
        else ops.gemm_w8a8(n8, sn, wg)
    torch.cuda.synchronize()
    lo, hi = int(bt.start[0]), int(bt.start[-1])
    (rq, qm), _, _, _ = _append_reference(bt, qkv, qnw, knw, cos, sin, nH * hd, (nH + nkv) * hd)
    _close16(q.view(bt.T, nH, hd)[lo:hi], rq[lo:hi], qm[lo:hi], "q")
    bt.check(o, q)
    _check(t, h, pfw, paw, 0.9, h1, n8, sn, "norm")
    ref = (n8.to(F64) @ wg.w8.to(F64)) * sn.to(F64)[:, None] * wg.sw8.to(F64)
    eps = torch.finfo(y.dtype).eps / 2 + 2.0 ** -22
    assert ((y.to(F64) - ref).abs() <= eps * ref.abs() + 2.0 ** -25).all()
    assert L.query(L.Q_KERNEL_STATUS) == 0


@pytest.mark.parametrize("D", [256, 3840, 40000])
def test_rows_that_are_not_finite(D):
    """A row with a NaN or an infinity: its residual, scale and codes are those of the three calls; the others' too."""
    h, x, w = torch.randn(5, D, device=DEV), torch.randn(5, D, device=DEV), 1 + 0.1 * torch.randn(D, device=DEV)
    x[1, 3], h[3, D - 1] = float("nan"), float("inf")
    h2, h0, x0 = h.clone(), h.clone(), x.clone()
    a8, sa = ops.rows_normadd_i8(x, h, w, w_post=w)
    ops.rows_normadd(x, w, h2, 1.0)
    b8, sb = ops.cast_i8(ops.rows_rmsnorm(h2, w))
    for r in (1, 3):
        assert torch.equal(torch.isfinite(h[r]), torch.isfinite(h2[r])) and not torch.isfinite(h[r]).all()
        assert torch.equal(a8[r], b8[r]) and sa[r] == sb[r]
    fine = [0, 2, 4]
    _check(x0[fine], h0[fine], w, w, 1.0, h[fine], a8[fine], sa[fine])


def test_captured_and_replayed():
    M, D = 37, 3840
    x, h, w = torch.randn(M, D, device=DEV).half(), torch.randn(M, D, device=DEV), 1 + 0.1 * torch.randn(D, device=DEV)
    out, a8, sa = torch.empty_like(h), torch.empty(M, D, dtype=torch.int8, device=DEV), torch.empty(M, device=DEV)
    ops.rows_normadd_i8(x, h, w, w_post=w, h_out=out, A8=a8, sa=sa)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.rows_normadd_i8(x, h, w, w_post=w, h_out=out, A8=a8, sa=sa)
    for k in range(3):
        h.mul_(-1.5)
        graph.replay()
        torch.cuda.synchronize()
        _check(x, h, w, w, 1.0, out, a8, sa)
        b8, sb = ops.rows_normadd_i8(x, h, w, w_post=w, h_out=torch.empty_like(h))
        assert torch.equal(a8, b8) and torch.equal(sa, sb)


@pytest.mark.parametrize("D", [256, 3840, 9600, 40000])
def test_rows_below_the_smallest_scale(D):
    """Rows whose largest magnitude is under 127e-12 have the scale 1e-12 and codes that are no longer spread over the whole
    range: h of 5e-14 has y of 5e-11 (eps alone makes the norm's factor 1000) and the code 50."""
    g = torch.Generator(device=DEV).manual_seed(D)
    size = torch.tensor([1e-20, 4e-16, 5e-14, 1e-13, 1.2e-13], device=DEV)
    h = (2 * torch.rand(5, D, generator=g, device=DEV) - 1) * size[:, None]
    h[:, 5] = size
    w = torch.ones(D, device=DEV)
    a8, sa = ops.rows_normadd_i8(None, h, w)
    assert (sa == np.float32(1e-12)).all()
    y = h.to(F64) * (h.to(F64).pow(2).mean(-1, keepdim=True) + 1e-6).rsqrt()
    code = y / 1e-12
    assert ((a8.to(F64) - code).abs() <= 0.5 + code.abs() * 2.0 ** -19).all()
    assert (a8[:2] == 0).all() and a8[2, 5] == 50 and a8[3, 5] == 100 and a8[4, 5] == 120


def test_large_values_and_zeros_each_by_itself():
    D = 256
    h = torch.zeros(4, D, device=DEV)
    h[1], h[2], h[3, 7] = 1e18, 1e-20, -1e15
    a8, sa = ops.rows_normadd_i8(torch.zeros(4, D, device=DEV), h, torch.ones(D, device=DEV))
    assert (a8[0] == 0).all() and (a8[1] == 127).all() and (a8[2] == 0).all()
    assert a8[3, 7] == -127 and (a8[3].abs().sum() == 127)
    assert sa[0] == np.float32(1e-12) and sa[2] == np.float32(1e-12)
    assert abs(sa[1].item() * 127 - 1) < 1e-5 and abs(sa[3].item() * 127 / 16 - 1) < 1e-5
