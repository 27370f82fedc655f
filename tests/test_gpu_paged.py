"""Batches over a paged KV cache (g4b_paged_plan, g4b_paged_append, g4b_paged_attn) against the definitions in
64 bits, computed with plain torch one sequence at a time.

Every cache starts as NaN; only the places that the batch may read hold numbers, so a value taken from behind a
mask, from another page or from a row that is not there shows at once.  Tolerances count roundings:
  append  an output is rounded to f16 once (2^-11 of its value, 2^-25 below the normal range); its f32 path
          makes under 16 roundings of terms no larger than |n cos| + |partner sin|: 2^-20 of that sum.
  attend  the output's rounding (2^-11 f16, 2^-24 f32), and on every weight: its own rounding to f16 (2^-11, where
          many rows share a tile), the exponential (2^-21), and twice the error of a score, which is at most
          hd 2^-23 of sum |q_i k_i| scale (f32 sums of exact products, truncated or rounded, in any order).  An error of d on
          every weight moves an output by at most 2 d sum_j p_j |v_j|."""
import numpy as np
import pytest
import torch

from g4b import _lib as L
from g4b import ops
from g4b.paged import PagedPlan

pytestmark = pytest.mark.gpu
DEV = "cuda"
F64 = torch.float64


class Batch:
    """A ragged batch: new[b] tokens for sequence b, total[b] held with them, `prefix` of those shared."""

    def __init__(self, nH, nkv, hd, page, new, total, prefix=0, window=0, seed=0, front=0, back=0, spare_pages=5,
                 prefix_pages=None):
        self.nH, self.nkv, self.hd, self.page, self.window, self.prefix = nH, nkv, hd, page, window, prefix
        self.new, self.total, self.B = list(new), list(total), len(new)
        self.start = np.concatenate([[0], np.cumsum(new)]).astype(np.int64) + front
        self.T = int(self.start[-1]) + back
        rng = np.random.default_rng(seed)
        self.pre_pages = -(-prefix // page) if prefix_pages is None else prefix_pages
        self.own_pages = max([1] + [-(-(t - prefix) // page) for t in total])
        self.pages = self.pre_pages + self.B * self.own_pages + spare_pages
        order = rng.permutation(self.pages).astype(np.int32)
        self.pre_ids = order[:self.pre_pages]
        self.ids = order[self.pre_pages:self.pre_pages + self.B * self.own_pages].reshape(self.B, self.own_pages)
        self.g = torch.Generator(device=DEV).manual_seed(seed)
        t32 = lambda a: torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(DEV)  # noqa: E731
        self.q_start, self.kv_len, self.table = t32(self.start), t32(self.total), t32(self.ids)
        self.prefix_table = t32(self.pre_ids) if self.pre_pages else None
        self.prefix_len = t32([prefix]) if self.pre_pages else None
        self.kc = torch.full((self.pages, nkv, page, hd), float("nan"), dtype=torch.float16, device=DEV)
        self.vc = torch.full_like(self.kc, float("nan"))

    def place(self, b, p):
        """(page, slot) of position p of sequence b."""
        if p < self.prefix:
            return int(self.pre_ids[p // self.page]), p % self.page
        return int(self.ids[b, (p - self.prefix) // self.page]), (p - self.prefix) % self.page

    def places(self, b, n):
        at = [self.place(b, p) for p in range(n)]
        return (torch.tensor([x[0] for x in at], dtype=torch.long, device=DEV),
                torch.tensor([x[1] for x in at], dtype=torch.long, device=DEV))

    def randn(self, *s, dtype=torch.float32):
        return torch.randn(*s, generator=self.g, device=DEV, dtype=dtype)

    def fill(self):
        """Numbers at every position that a token may see."""
        done = 0
        for b in sorted(range(self.B), key=lambda b: -self.total[b]):
            n = self.total[b]
            lo = min(done, self.prefix)       # the longest sequence fills the prefix
            pg, sl = self.places(b, n)
            pg, sl = pg[lo:], sl[lo:]
            self.kc[pg, :, sl] = self.randn(len(pg), self.nkv, self.hd, dtype=torch.float16)
            self.vc[pg, :, sl] = self.randn(len(pg), self.nkv, self.hd, dtype=torch.float16)
            done = max(done, min(n, self.prefix))
        return self

    def queries(self, std=4.0):
        return self.randn(self.T, self.nH * self.hd, dtype=torch.float16) * (std * self.hd ** -0.5)

    def plan(self, T=None):
        p = PagedPlan(self.T, self.B, self.nH, self.nkv, self.hd, self.page, self.own_pages, self.pre_pages,
                      self.window, DEV)
        p.update(self.q_start, self.kv_len, self.prefix_len)
        return p

    def reference(self, q, scale=1.0, bad_pages=()):
        """(out, tolerance without the output's rounding) [T, nH, hd] in 64 bits; padding rows are NaN."""
        out = torch.full((self.T, self.nH, self.hd), float("nan"), dtype=F64, device=DEV)
        tol = torch.zeros_like(out)
        G = self.nH // self.nkv
        for b in range(self.B):
            n, t0, total = self.new[b], int(self.start[b]), self.total[b]
            if n == 0:
                continue
            pg, sl = self.places(b, total)
            k, v = self.kc[pg, :, sl].to(F64), self.vc[pg, :, sl].to(F64)      # [total, nkv, hd]
            j = torch.arange(total, device=DEV)
            there = torch.ones(total, dtype=torch.bool, device=DEV)
            for x in bad_pages:
                there &= pg != x
            for i0 in range(0, n, 128):
                m = min(128, n - i0)
                pos = torch.arange(total - n + i0, total - n + i0 + m, device=DEV)
                see = (j[None] <= pos[:, None]) & there[None]
                if self.window:
                    see &= j[None] > pos[:, None] - self.window
                qq = q[t0 + i0:t0 + i0 + m].to(F64).view(m, self.nkv, G, self.hd)
                used = see.any(0)
                kk = torch.where(used[:, None, None], k, torch.zeros_like(k))
                vv = torch.where(used[:, None, None], v, torch.zeros_like(v))
                s = torch.einsum("mkgd,jkd->mkgj", qq, kk) * scale
                s = torch.where(see[:, None, None], s, torch.full_like(s, float("-inf")))
                top = s.amax(-1, keepdim=True) if total else s.new_zeros(m, self.nkv, G, 1)
                p = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
                den = p.sum(-1, keepdim=True)
                p = p / torch.where(den == 0, torch.ones_like(den), den)
                mag = torch.einsum("mkgd,jkd->mkgj", qq.abs(), kk.abs()) * scale
                mag = torch.where(see[:, None, None], mag, torch.zeros_like(mag)).amax(-1, keepdim=True) if total else 0
                d = 2.0 ** -11 + 2.0 ** -21 + 2 * self.hd * 2.0 ** -23 * mag
                o = torch.einsum("mkgj,jkd->mkgd", p, vv)
                a = torch.einsum("mkgj,jkd->mkgd", p, vv.abs())
                out[t0 + i0:t0 + i0 + m] = o.reshape(m, self.nH, self.hd)
                tol[t0 + i0:t0 + i0 + m] = (2 * d * a).reshape(m, self.nH, self.hd)
        return out, tol

    def check(self, got, q, scale=1.0, bad_pages=()):
        ref, tol = self.reference(q, scale, bad_pages)
        got64 = got.to(F64).view(self.T, self.nH, self.hd)
        eps = torch.finfo(got.dtype).eps / 2
        lo, hi = int(self.start[0]), int(self.start[-1])
        err = (got64 - ref).abs()[lo:hi]
        lim = (tol + eps * ref.abs() + 2.0 ** -25)[lo:hi]
        assert bool(torch.isfinite(got64[lo:hi]).all())
        worst = (err - lim).max().item() if err.numel() else 0.0
        assert worst <= 0, f"off by {err.max().item():.3e}, {(err / lim).max().item():.2f} of the tolerance"
        assert L.query(L.Q_KERNEL_STATUS) == 0


def _attend(bt, q, plan=None, out_dtype=torch.float16, scale=1.0, out=None):
    plan = plan or bt.plan()
    if out is None:
        out = torch.full((bt.T, bt.nH * bt.hd), 7.0, dtype=out_dtype, device=DEV)
    plan.attend(q, bt.kc, bt.vc, bt.table, bt.prefix_table, out=out, scale=scale)
    torch.cuda.synchronize()
    return out


HEADS = [(16, 8, 256), (8, 1, 128), (4, 2, 512), (6, 2, 128), (3, 3, 256), (16, 1, 512)]


@pytest.mark.parametrize("nH,nkv,hd", HEADS)
@pytest.mark.parametrize("page,new,total,prefix,window", [
    (64, [1], [1], 0, 0),                                     # one token, one key
    (64, [1], [700], 0, 0),
    (16, [1, 1, 1], [5, 64, 65], 0, 0),
    (32, [1, 1, 1, 1], [130, 101, 377, 102], 100, 0),         # the prefix ends inside a page
    (128, [1] * 9, [200 + 37 * i for i in range(9)], 150, 64),  # a window that begins in the prefix for some only
    (64, [2, 1, 4, 3], [300, 260, 259, 500], 256, 0),         # a few proposed tokens each
])
def test_decode_batches(nH, nkv, hd, page, new, total, prefix, window):
    bt = Batch(nH, nkv, hd, page, new, total, prefix, window, seed=hd + nH).fill()
    q = bt.queries()
    bt.check(_attend(bt, q), q)


@pytest.mark.parametrize("nH,nkv,hd", HEADS)
@pytest.mark.parametrize("page,new,total,prefix,window", [
    (64, [70], [70], 0, 0),                                   # a first prompt
    (16, [33, 90], [40, 333], 0, 0),
    (32, [130, 17, 1], [400, 217, 260], 200, 0),              # chunks behind a prefix, and a decode among them
    (64, [150, 60], [391, 460], 230, 100),                    # window
    (128, [65], [1300], 0, 129),
])
def test_prompt_chunks(nH, nkv, hd, page, new, total, prefix, window):
    bt = Batch(nH, nkv, hd, page, new, total, prefix, window, seed=hd + page).fill()
    q = bt.queries()
    bt.check(_attend(bt, q), q)


@pytest.mark.parametrize("nH,nkv,hd", [(16, 8, 256), (8, 1, 128)])
def test_long_ragged_batch_over_a_prefix(nH, nkv, hd):
    rng = np.random.default_rng(3)
    new = [1] * 70
    total = [5000 + int(x) for x in rng.integers(1, 900, 70)]
    bt = Batch(nH, nkv, hd, 64, new, total, prefix=5000, seed=1).fill()
    q = bt.queries()
    bt.check(_attend(bt, q), q)


@pytest.mark.parametrize("hd,nH,nkv", [(256, 16, 8), (512, 4, 2)])
def test_f32_output_scale_and_strides(hd, nH, nkv):
    bt = Batch(nH, nkv, hd, 32, [1, 40, 3], [90, 140, 33], 30, seed=5, back=2).fill()
    wide = bt.randn(bt.T, nH * hd + 24, dtype=torch.float16)
    q = wide[:, 8:8 + nH * hd]
    out = torch.full((bt.T, nH * hd + 16), 7.0, dtype=torch.float32, device=DEV)
    view = out[:, 8:8 + nH * hd]
    _attend(bt, q, out=view, scale=hd ** -0.5)
    bt.check(view, q, scale=hd ** -0.5)
    assert (out[:, :8] == 7).all() and (out[:, 8 + nH * hd:] == 7).all() and (view[-2:] == 7).all()


def test_rows_outside_the_sequences_are_left():
    bt = Batch(16, 8, 256, 64, [1, 0, 20, 0], [65, 10, 90, 0], 0, seed=6, front=3, back=4).fill()
    q = bt.queries()
    out = _attend(bt, q)
    bt.check(out, q)
    assert (out[:3] == 7).all() and (out[-4:] == 7).all()


@pytest.mark.parametrize("hd,nH,nkv", [(256, 16, 8), (512, 4, 2)])
def test_tokens_without_keys_give_zeros(hd, nH, nkv):
    """More new tokens than the length says (positions below 0), and a sequence whose only pages are not there."""
    bt = Batch(nH, nkv, hd, 16, [1, 1, 2], [20, 16, 40], 0, seed=7).fill()
    bt.table[1, 0] = -1                                  # all of sequence 1's keys
    bt.kv_len[2] = 1                                     # its first token has position -1
    q = bt.queries()
    out = _attend(bt, q).view(bt.T, nH, hd)
    assert (out[1] == 0).all() and (out[2] == 0).all()
    bt.total[2], bt.new[2] = 1, 1
    bt.start[2] = 3
    ref, _ = bt.reference(q)                             # token 3 sees its one key
    assert (out[3].to(F64) - ref[3]).abs().max() < 1e-2
    bt.total[1] = 0
    assert L.query(L.Q_KERNEL_STATUS) == 0


@pytest.mark.parametrize("hd,nH,nkv,new", [(256, 16, 8, [1, 1]), (128, 8, 1, [20, 3]), (512, 4, 2, [5, 2])])
@pytest.mark.parametrize("bad", [-1, 10**9, None])
def test_pages_that_are_not_there(hd, nH, nkv, new, bad):
    bt = Batch(nH, nkv, hd, 16, new, [150, 120], 50, seed=8).fill()
    q = bt.queries()
    gone = [int(bt.ids[0, 1]), int(bt.ids[1, 3]), int(bt.pre_ids[1])]
    bad = bt.pages if bad is None else bad               # the first id that is too large
    bt.table[0, 1] = bad
    bt.table[1, 3] = bad
    bt.prefix_table[1] = bad
    bt.check(_attend(bt, q), q, bad_pages=gone)


def test_prefix_of_length_zero_and_short_sequences():
    """Prefix pages with a prefix of no token; a sequence that ends inside the prefix."""
    bt = Batch(16, 8, 256, 32, [1, 3], [70, 41], 0, seed=9, prefix_pages=4).fill()
    q = bt.queries()
    bt.check(_attend(bt, q), q)
    bt = Batch(16, 8, 256, 32, [1, 3, 2], [170, 41, 1 + 100], 100, seed=9).fill()
    q = bt.queries()
    bt.check(_attend(bt, q), q)


@pytest.mark.parametrize("hd,nH,nkv,new", [(256, 16, 8, 4), (512, 4, 2, 3), (128, 8, 1, 2), (256, 16, 8, 30), (128, 8, 1, 40)])
def test_values_behind_the_mask_do_not_reach_a_row(hd, nH, nkv, new):
    """The last token's key and value are infinite: the tokens before it must not notice."""
    bt = Batch(nH, nkv, hd, 16, [new, 1], [new + 21, 50], 0, seed=10).fill()
    q = bt.queries()
    clean = _attend(bt, q).clone()
    pg, sl = bt.place(0, new + 20)
    bt.kc[pg, :, sl] = float("inf")
    bt.vc[pg, :, sl] = float("-inf")
    out = _attend(bt, q)
    assert torch.equal(out[:new - 1], clean[:new - 1]) and torch.equal(out[new:], clean[new:])
    assert not torch.isfinite(out[new - 1]).any()


def test_scores_of_the_lowest_values():
    """Scores near the largest negative finite ones still give weights; equal scores give equal weights."""
    bt = Batch(16, 8, 256, 64, [1], [300], 0, seed=11).fill()
    q = bt.queries()
    bt.kc.copy_(torch.where(torch.isnan(bt.kc), bt.kc, torch.full_like(bt.kc, -60000.0)))
    q.copy_(torch.full_like(q, 200.0))
    out = _attend(bt, q)
    pg, sl = bt.places(0, 300)
    mean = bt.vc[pg, :, sl].to(F64).mean(0).repeat_interleave(2, 0)
    a = bt.vc[pg, :, sl].to(F64).abs().mean(0).repeat_interleave(2, 0)
    assert ((out.view(16, 256).to(F64) - mean).abs() <= 2.0 ** -11 * mean.abs() + 2 * (2.0 ** -11 + 2.0 ** -20) * a).all()


def test_lengths_that_lie_stay_inside_the_buffers():
    """Starts that fall and run past T, lengths past the tables: cut as the header says, no row outside is touched."""
    bt = Batch(16, 8, 256, 16, [2, 3, 1], [40, 33, 48], 0, seed=12, back=2).fill()
    bt.kc.nan_to_num_(0.5)
    bt.vc.nan_to_num_(0.5)
    q = bt.queries()
    bt.q_start.copy_(torch.tensor([-5, 4, 1, 9999], dtype=torch.int32))
    bt.kv_len.copy_(torch.tensor([-3, 10**9, 2**31 - 1], dtype=torch.int32))
    out = _attend(bt, q)
    assert torch.isfinite(out).all() and L.query(L.Q_KERNEL_STATUS) == 0
    assert (out[:4] == 0).all()                          # sequence 0: no key
    # sequence 2 has rows 4.. of all T, its length cut to its three pages
    bt.start, bt.new, bt.total = np.array([0, 4, 4, bt.T]), [4, 0, bt.T - 4], [0, 48, 48]
    ref, tol = bt.reference(q)
    err = (out.view(bt.T, 16, 256).to(F64) - ref)[4:].abs()
    assert (err <= tol[4:] + 2.0 ** -11 * ref[4:].abs() + 2.0 ** -25).all()


def test_a_plan_of_other_sizes_writes_nothing():
    bt = Batch(16, 8, 256, 64, [1, 1], [65, 90], 0, seed=13).fill()
    q = bt.queries()
    plan = PagedPlan(bt.T, bt.B, 16, 8, 256, 64, bt.own_pages, 0, 0, DEV)    # never updated
    out = torch.full((bt.T, 4096), 7.0, dtype=torch.float16, device=DEV)
    plan.attend(q, bt.kc, bt.vc, bt.table, out=out)
    torch.cuda.synchronize()
    assert (out == 7).all()
    assert L.query(L.Q_KERNEL_STATUS) == 2 and L.query(L.Q_KERNEL_STATUS) == 0
    other = Batch(16, 8, 256, 64, [1, 1, 1], [65, 90, 4], 0, seed=13)
    plan._plan = torch.cat((other.plan()._plan, torch.zeros(1 << 20, dtype=torch.uint8, device=DEV)))
    qkv = bt.randn(bt.T, 8192)
    kc = bt.kc.clone()
    w = torch.ones(256, device=DEV)
    rot = torch.ones(bt.own_pages * 64, 256, device=DEV)
    plan.append(qkv, w, w, rot, rot, bt.kc, bt.vc, bt.table, 4096, 6144, q_out=out)
    torch.cuda.synchronize()
    assert (out == 7).all() and torch.equal(bt.kc.view(torch.int16), kc.view(torch.int16))
    assert L.query(L.Q_KERNEL_STATUS) == 2


def test_python_refusals():
    bt = Batch(16, 8, 256, 64, [1, 1], [65, 90], 0, seed=13).fill()
    plan, q = bt.plan(), bt.queries()
    with pytest.raises(ValueError):
        plan.attend(q, bt.kc, bt.vc, bt.table, prefix_table=bt.table[0])
    with pytest.raises(ValueError):
        plan.attend(q.float(), bt.kc, bt.vc, bt.table)
    with pytest.raises(ValueError):
        plan.attend(q[:1], bt.kc, bt.vc, bt.table)
    with pytest.raises(ValueError):
        plan.attend(q, bt.kc[:, :, :32], bt.vc[:, :, :32], bt.table)
    with pytest.raises(ValueError):
        plan.attend(q, bt.kc.cpu(), bt.vc, bt.table)
    with pytest.raises(ValueError):
        plan.update(bt.q_start[:2], bt.kv_len)
    with pytest.raises(L.G4BError):
        PagedPlan(1, 1, 16, 8, 96, 64, 1)


def _append_reference(bt, qkv, qnw, knw, cos, sin, koff, voff):
    """(value, magnitude of the rotation's terms) of q [T, nH, hd], k and v [T, nkv, hd], positions [T]."""
    pos = torch.full((bt.T,), -1, dtype=torch.long, device=DEV)
    for b in range(bt.B):
        s, n = int(bt.start[b]), bt.new[b]
        pos[s:s + n] = torch.arange(bt.total[b] - n, bt.total[b], device=DEV)
    x = qkv.to(F64)
    c, s = cos[pos.clamp(min=0)].to(F64)[:, None], sin[pos.clamp(min=0)].to(F64)[:, None]

    def normed(off, heads):
        y = x[:, off:off + heads * bt.hd].reshape(bt.T, heads, bt.hd)
        return y * (y.pow(2).mean(-1, keepdim=True) + 1e-6).rsqrt()

    def turn(y):
        h = bt.hd // 2
        o = torch.cat((-y[..., h:], y[..., :h]), -1)
        return y * c + o * s, (y * c).abs() + (o * s).abs()

    v = normed(voff, bt.nkv)
    return turn(normed(0, bt.nH) * qnw.to(F64)), turn(normed(koff, bt.nkv) * knw.to(F64)), (v, v.abs()), pos


def _close16(got, ref, mag, what):
    lim = 2.0 ** -11 * ref.abs() + 2.0 ** -20 * mag + 2.0 ** -25
    err = (got.to(F64) - ref).abs()
    assert (err <= lim).all(), f"{what}: {(err / lim).max().item():.2f} of the tolerance"


@pytest.mark.parametrize("nH,nkv,hd", HEADS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("page,new,total,prefix,keqv", [
    (64, [1], [1], 0, False),
    (16, [1, 0, 1, 2], [33, 7, 50, 49], 32, False),
    (32, [1, 1, 1], [131, 129, 140], 128, True),
    (128, [300, 5, 90], [311, 77, 90], 0, False),
    (64, [20, 40], [30, 45], 25, False),                      # the first chunk begins inside the prefix: not written there
])
def test_append(nH, nkv, hd, dtype, page, new, total, prefix, keqv):
    bt = Batch(nH, nkv, hd, page, new, total, prefix, seed=hd + page + nH, front=1, back=2)
    nq, nk = nH * hd, nkv * hd
    koff, voff = nq, nq if keqv else nq + nk
    wide = (bt.randn(bt.T, nq + 2 * nk + 16) * torch.exp(bt.randn(bt.T, 1))).to(dtype)
    qkv = wide[:, 8:]
    if qkv.data_ptr() % 16:
        qkv = wide[:, :-16]
    qnw, knw = 1 + 0.2 * bt.randn(hd), 1 + 0.2 * bt.randn(hd)
    n_pos = (bt.own_pages + bt.pre_pages) * page
    inv = 10000.0 ** (-torch.arange(0, hd, 2, device=DEV, dtype=F64) / hd)
    ang = torch.arange(n_pos, device=DEV, dtype=F64)[:, None] * torch.cat((inv, inv))
    cos, sin = ang.cos().float(), ang.sin().float()
    q_out = torch.full((bt.T, nq), 7.0, dtype=torch.float16, device=DEV)
    bt.plan().append(qkv, qnw, knw, cos, sin, bt.kc, bt.vc, bt.table, koff, voff, q_out=q_out)
    torch.cuda.synchronize()
    (q, qm), (k, km), (v, vm), pos = _append_reference(bt, qkv, qnw, knw, cos, sin, koff, voff)
    lo, hi = int(bt.start[0]), int(bt.start[-1])
    _close16(q_out.view(bt.T, nH, hd)[lo:hi], q[lo:hi], qm[lo:hi], "q")
    assert (q_out[:lo] == 7).all() and (q_out[hi:] == 7).all()
    written = torch.zeros(bt.pages, page, dtype=torch.bool, device=DEV)
    for b in range(bt.B):
        for i in range(new[b]):
            t = int(bt.start[b]) + i
            p = int(pos[t])
            if p < prefix:
                continue
            pg, sl = bt.place(b, p)
            written[pg, sl] = True
            _close16(bt.kc[pg, :, sl], k[t], km[t], "k")
            _close16(bt.vc[pg, :, sl], v[t], vm[t], "v")
    for c in (bt.kc, bt.vc):
        kept = c.permute(0, 2, 1, 3)[~written]
        assert torch.isnan(kept).all()                       # every other place as it was
    assert L.query(L.Q_KERNEL_STATUS) == 0


def test_append_skips_pages_that_are_not_there():
    bt = Batch(16, 8, 256, 16, [20, 1], [20, 5], 0, seed=20)
    bt.table[0, 0] = -7
    bt.table[1, 0] = bt.pages
    w, rot = torch.ones(256, device=DEV), torch.ones(bt.own_pages * 16, 256, device=DEV)
    bt.plan().append(bt.randn(bt.T, 8192), w, w, rot, rot, bt.kc, bt.vc, bt.table, 4096, 6144)
    torch.cuda.synchronize()
    pg, _ = bt.place(0, 16)
    mask = torch.ones(bt.pages, dtype=torch.bool, device=DEV)
    mask[pg] = False
    assert torch.isnan(bt.kc[mask]).all() and torch.isfinite(bt.kc[pg, :, :4]).all() and torch.isnan(bt.kc[pg, :, 4:]).all()
    assert L.query(L.Q_KERNEL_STATUS) == 0


def test_caches_past_two_to_the_31_elements():
    nkv, hd, page = 8, 256, 64
    pages = (1 << 31) // (nkv * hd * page) + 3
    bt = Batch(16, nkv, hd, page, [1, 30], [100, 64], 0, seed=21)
    kc = torch.zeros(pages, nkv, page, hd, dtype=torch.float16, device=DEV)
    vc = torch.zeros_like(kc)
    last = list(range(pages - bt.B * bt.own_pages, pages))
    bt.ids = np.array(last[::-1], dtype=np.int32).reshape(bt.B, bt.own_pages)
    bt.table.copy_(torch.from_numpy(bt.ids))
    bt.kc, bt.vc, bt.pages = kc, vc, pages
    bt.fill()
    q = bt.queries()
    bt.check(_attend(bt, q), q)
    w, rot = torch.ones(256, device=DEV), torch.ones(bt.own_pages * page, 256, device=DEV)
    before = kc[:64].clone()
    bt.plan().append(bt.randn(bt.T, 8192), w, w, rot, rot, kc, vc, bt.table, 4096, 6144)
    pg, sl = bt.place(0, 99)
    assert (kc[pg, :, sl] != 0).any() and torch.equal(kc[:64], before)


def test_graph_replays_follow_the_lengths():
    bt = Batch(16, 8, 256, 64, [1, 1, 1], [100, 300, 161], 64, seed=22).fill()
    q = bt.queries()
    plan = bt.plan()
    out = torch.full((bt.T, 4096), 7.0, dtype=torch.float16, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        plan.update(bt.q_start, bt.kv_len, bt.prefix_len)
        plan.attend(q, bt.kc, bt.vc, bt.table, bt.prefix_table, out=out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.update(bt.q_start, bt.kv_len, bt.prefix_len)
        plan.attend(q, bt.kc, bt.vc, bt.table, bt.prefix_table, out=out)
    for total in ([100, 300, 161], [65, 140, 161], [64, 299, 90]):
        bt.kv_len.copy_(torch.tensor(total, dtype=torch.int32))
        bt.total = total
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        bt.check(out, q)


def test_two_plans_at_once_on_two_streams():
    a = Batch(16, 8, 256, 64, [1] * 40, [2000 + i for i in range(40)], 1900, seed=23).fill()
    b = Batch(8, 1, 128, 16, [60, 1, 5], [900, 700, 300], 200, seed=24).fill()
    qa, qb = a.queries(), b.queries()
    pa, pb = a.plan(), b.plan()
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = []
    for _ in range(4):
        oa = pa.attend(qa, a.kc, a.vc, a.table, a.prefix_table, stream=sa)
        ob = pb.attend(qb, b.kc, b.vc, b.table, b.prefix_table, stream=sb)
        outs.append((oa, ob))
    torch.cuda.synchronize()
    for oa, ob in outs:
        a.check(oa, qa)
        b.check(ob, qb)
        assert torch.equal(oa, outs[0][0]) and torch.equal(ob, outs[0][1])    # the same bits every time


@pytest.mark.parametrize("nH,nkv,hd,new", [(16, 8, 256, 3), (16, 8, 256, 40), (4, 2, 512, 40), (8, 1, 128, 90)])
def test_widest_windows_and_positions_below_zero(nH, nkv, hd, new):
    """A window of 2^31 - 1 keys is none, before a sequence's first position too."""
    outs = []
    for window in (0, 2**31 - 1):
        bt = Batch(nH, nkv, hd, 16, [new, 1], [new, 50], 0, window, seed=30).fill()
        bt.kv_len[0] = new - 2
        outs.append(_attend(bt, bt.queries()))
    assert torch.equal(outs[0], outs[1]) and (outs[0][:2] == 0).all() and (outs[0][2:] != 0).any(-1).all()


@pytest.mark.parametrize("prefix", [0, 40])
def test_as_many_sequences_as_a_plan_takes(prefix):
    rng = np.random.default_rng(5)
    new = rng.integers(0, 3, 4096)
    total = new + prefix + rng.integers(0, 20, 4096)
    bt = Batch(2, 1, 128, 16, new, total, prefix, seed=31).fill()
    q = bt.queries()
    bt.check(_attend(bt, q), q)


def test_sequences_that_share_a_page():
    bt = Batch(16, 8, 256, 32, [1, 2, 20], [70, 66, 90], 0, seed=32)
    bt.ids[1:, :2] = bt.ids[0, :2]
    bt.table.copy_(torch.from_numpy(bt.ids))
    bt.fill()
    q = bt.queries()
    bt.check(_attend(bt, q), q)


def test_queries_and_results_in_one_buffer():
    bt = Batch(16, 8, 256, 32, [1, 40, 3], [90, 140, 33], 30, seed=33).fill()
    wide = torch.cat((bt.queries(), torch.full((bt.T, 4096), 7.0, dtype=torch.float16, device=DEV)), 1)
    q, out = wide[:, :4096], wide[:, 4096:]
    before = q.clone()
    bt.check(_attend(bt, q, out=out), before)
    assert torch.equal(q, before)
    with pytest.raises(L.G4BError):
        _attend(bt, q, out=q)


def test_a_plan_made_while_its_stream_is_busy():
    """What the constructor queues on its own stream is done before another stream's calls."""
    bt = Batch(16, 8, 256, 64, [1, 1], [65, 90], 0, seed=34).fill()
    q, side = bt.queries(), torch.cuda.Stream()
    out = torch.full((bt.T, 4096), 7.0, dtype=torch.float16, device=DEV)
    torch.cuda.synchronize()
    torch.cuda._sleep(100_000_000)                           # some 50 ms
    plan = PagedPlan(bt.T, bt.B, 16, 8, 256, 64, bt.own_pages, 0, 0, DEV)
    plan.update(bt.q_start, bt.kv_len, stream=side)
    plan.attend(q, bt.kc, bt.vc, bt.table, out=out, stream=side)
    torch.cuda.synchronize()
    bt.check(out, q)


def test_a_plan_dropped_while_another_stream_works_with_it():
    """Its memory serves nothing else before that work is done."""
    bt = Batch(16, 8, 256, 64, [1] * 30, [900 + i for i in range(30)], 800, seed=35).fill()
    q, side = bt.queries(), torch.cuda.Stream()
    plan = bt.plan()
    out = torch.full((bt.T, 4096), 7.0, dtype=torch.float16, device=DEV)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(50_000_000)
        plan.attend(q, bt.kc, bt.vc, bt.table, bt.prefix_table, out=out)
    sizes = plan._plan.numel(), plan._ws.numel()
    del plan
    other = [torch.zeros(n, dtype=torch.uint8, device=DEV) for n in sizes]
    torch.cuda.synchronize()
    bt.check(out, q)
    assert all((x == 0).all() for x in other)


def test_two_threads_with_other_sizes():
    """Calls of two host threads whose kernels need different amounts of shared memory."""
    import threading

    cases = [Batch(4, 2, 256, 16, [150, 150], [150, 150], 0, seed=36),
             Batch(16, 8, 256, 16, [300] + [0] * 500, [300] * 501, 0, seed=37)]
    jobs, errors = [], []
    for bt in cases:
        nq, nk = bt.nH * bt.hd, bt.nkv * bt.hd
        w, rot = torch.ones(bt.hd, device=DEV), torch.ones(bt.own_pages * 16, bt.hd, device=DEV)
        args = (bt.randn(bt.T, nq + 2 * nk), w, w, rot, rot, bt.kc, bt.vc, bt.table, nq, nq + nk)
        jobs.append((bt, bt.plan(), args, torch.cuda.Stream()))
    torch.cuda.synchronize()

    def run(bt, plan, args, stream):
        try:
            for _ in range(200):
                plan.update(bt.q_start, bt.kv_len, stream=stream)
                plan.append(*args, stream=stream)
        except Exception as e:                               # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=run, args=j) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors
    for bt, _, _, _ in jobs:
        pg, sl = bt.places(0, bt.total[0])
        assert torch.isfinite(bt.kc[pg, :, sl]).all() and torch.isfinite(bt.vc[pg, :, sl]).all()


@pytest.mark.parametrize("T,hd,nH,nkv", [(6, 256, 16, 8), (320, 128, 8, 1)])
def test_a_captured_step_of_append_and_attention(T, hd, nH, nkv):
    """Plan, append, attention in one graph, replayed while the sequences grow: the bits of eager calls."""
    n = T // 2
    a, b = (Batch(nH, nkv, hd, 32, [n, n], [400, 400], 20, seed=38) for _ in range(2))
    nq, nk = nH * hd, nkv * hd
    qkv = a.randn(a.T, nq + 2 * nk)
    w = 1 + 0.1 * a.randn(hd)
    rot = a.randn((a.own_pages + a.pre_pages) * 32, hd)
    for bt in (a, b):
        for c in (bt.kc, bt.vc):
            c.copy_(torch.linspace(-1, 1, c.numel(), device=DEV).half().view(c.shape))
    out = [torch.empty(a.T, nq, dtype=torch.float16, device=DEV) for _ in range(2)]

    def step(bt, plan, o):
        plan.update(bt.q_start, bt.kv_len, bt.prefix_len)
        q = plan.append(qkv, w, w, rot, rot, bt.kc, bt.vc, bt.table, nq, nq + nk)
        plan.attend(q, bt.kc, bt.vc, bt.table, bt.prefix_table, out=o)

    plans = [a.plan(), b.plan()]
    step(a, plans[0], out[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(a, plans[0], out[0])
    for k, total in enumerate(([n + 20, n + 21], [n + 40, n + 20], [n + 100, n + 190])):
        for bt in (a, b):
            bt.kv_len.copy_(torch.tensor(total, dtype=torch.int32))
        qkv.mul_(1.5 - k)
        graph.replay()
        if k == 0:                                           # the eager and the warm-up call wrote a's pages only
            step(b, plans[1], out[1])
            b.kc.copy_(a.kc)
            b.vc.copy_(a.vc)
        step(b, plans[1], out[1])
        torch.cuda.synchronize()
        if k:
            assert torch.equal(out[0], out[1]) and torch.equal(a.kc, b.kc) and torch.equal(a.vc, b.vc)
    assert L.query(L.Q_KERNEL_STATUS) == 0


@pytest.mark.parametrize("nH,nkv,hd", HEADS)
@pytest.mark.parametrize("new,total,prefix", [
    ([1] * 64, [400 + 9 * i for i in range(64)], 300),        # joins of single rows and of small groups
    ([1] * 200, [301 + i for i in range(200)], 300),
    ([16] * 30, [2000] * 30, 0),
    ([150, 400, 1, 0, 33], [900, 1000, 801, 5, 833], 800),    # and of tiles of 128 rows
])
def test_plan_and_workspace_stay_inside_their_bytes(nH, nkv, hd, new, total, prefix):
    bt = Batch(nH, nkv, hd, 32, new, total, prefix, seed=40).fill()
    q, plan = bt.queries(), bt.plan()
    guarded = []
    for name in ("_plan", "_ws"):
        n = getattr(plan, name).numel()
        room = torch.full((n + 65536,), 0xA5, dtype=torch.uint8, device=DEV)
        setattr(plan, name, room[:n])
        setattr(plan, name + "_ptr", room.data_ptr())
        guarded.append((room, n))
    plan.update(bt.q_start, bt.kv_len, bt.prefix_len)
    bt.check(_attend(bt, q, plan), q)
    for room, n in guarded:
        assert (room[n:] == 0xA5).all()


@pytest.mark.parametrize("nH,nkv,hd,new", [(16, 8, 256, 4), (4, 2, 512, 3), (8, 1, 128, 2), (16, 8, 256, 70), (16, 1, 512, 20),
                                           (8, 1, 128, 40)])
@pytest.mark.parametrize("prefix", [0, 50])
def test_values_before_the_window_do_not_reach_a_row(nH, nkv, hd, new, prefix):
    """A key and value that are not finite, at the one position that only the first token's window still holds."""
    window = 20
    bt = Batch(nH, nkv, hd, 16, [new, 1], [new + 60, 90], prefix, window, seed=41).fill()
    q = bt.queries()
    clean = _attend(bt, q).clone()
    bt.check(clean, q)
    pg, sl = bt.place(0, 60 - window + 1)
    assert prefix == 0 or 60 - window + 1 < prefix
    bt.kc[pg, :, sl] = float("inf")
    bt.vc[pg, :, sl] = float("nan")
    out = _attend(bt, q)
    assert torch.equal(out[1:], clean[1:]) and not torch.isfinite(out[0]).any()


LONG = [(16, 8, 256, 0, torch.float16), (16, 8, 256, 1000, torch.float32), (8, 1, 128, 0, torch.float32),
        (8, 1, 128, 1000, torch.float16), (4, 2, 512, 0, torch.float16)]


@pytest.mark.parametrize("nH,nkv,hd,prefix,dtype", LONG)
def test_long_prompts_give_every_cta_many_tiles(nH, nkv, hd, prefix, dtype):
    """Several tiles a CTA, of several units each, the result of one read out while the next one's first products are
    made: against the definition, and the same bits every time beside a stream that keeps the memory busy."""
    bt = Batch(nH, nkv, hd, 64, [4096, 4096], [prefix + 4096, prefix + 4096], prefix, seed=50).fill()
    q, plan = bt.queries(), bt.plan()
    first = _attend(bt, q, plan, dtype)
    bt.check(first, q)
    side, a = torch.cuda.Stream(), torch.empty(1 << 28, dtype=torch.uint8, device=DEV)
    b, outs = torch.empty_like(a), [torch.empty_like(first) for _ in range(10)]
    torch.cuda.synchronize()
    for _ in range(20):
        with torch.cuda.stream(side):
            for _ in range(40):
                b.copy_(a)
        for o in outs:
            o.fill_(7.0)
            plan.attend(q, bt.kc, bt.vc, bt.table, bt.prefix_table, out=o)
        torch.cuda.synchronize()
        assert all(torch.equal(o, first) for o in outs)
    assert L.query(L.Q_KERNEL_STATUS) == 0


@pytest.mark.parametrize("nH,nkv,hd", [(16, 8, 256), (8, 1, 128), (4, 2, 512)])
def test_values_outside_the_window_of_many_tiles(nH, nkv, hd):
    """Infinite values every 500 positions, which only some rows of a tile see, in its first unit too: a row that sees
    none has the bits that it has without them."""
    n, window = 4096, 150
    bt = Batch(nH, nkv, hd, 32, [n, n], [n, n], 0, window, seed=51).fill()
    q, plan = bt.queries(), bt.plan()
    clean = _attend(bt, q, plan)
    bt.check(clean, q)
    at = torch.arange(250, n, 500, device=DEV)
    for b in range(2):
        pg, sl = bt.places(b, n)
        bt.vc[pg[at], :, sl[at]] = float("inf")
    pos = torch.arange(n, device=DEV)
    sees = ((at <= pos[:, None]) & (at > pos[:, None] - window)).any(1).repeat(2)
    for _ in range(20):
        out = _attend(bt, q, plan)
        assert torch.equal(out[~sees], clean[~sees]) and not torch.isfinite(out[sees]).any()


def test_a_plan_of_sizes_whose_hash_was_the_same():
    """Two batches that differ in tokens, sequences and tables: neither call takes the other's plan."""
    def made(T, table, prefix):
        return PagedPlan(T, T, 16, 8, 256, 64, table, prefix, 1024, DEV)

    t32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    for mine, other in (((67, 29, 16), (128, 12, 32)), ((128, 12, 32), (67, 29, 16))):
        plan, wrong = made(*mine), made(*other)
        n = other[0]
        wrong.update(torch.arange(n + 1, dtype=torch.int32, device=DEV), t32(*[1100] * n), t32(1000))
        room = torch.zeros(plan._plan.numel() + wrong._plan.numel(), dtype=torch.uint8, device=DEV)
        room[:wrong._plan.numel()] = wrong._plan
        plan._plan, plan._plan_ptr = room, room.data_ptr()
        T, table, prefix = mine
        kc = torch.zeros(prefix + T * table, 8, 64, 256, dtype=torch.float16, device=DEV)
        vc = torch.zeros_like(kc)
        ids = torch.arange(prefix, prefix + T * table, dtype=torch.int32, device=DEV).view(T, table)
        pre = torch.arange(prefix, dtype=torch.int32, device=DEV)
        out = torch.full((T, 4096), 7.0, dtype=torch.float16, device=DEV)
        q, w = torch.ones_like(out), torch.ones(256, device=DEV)
        rot = torch.ones((table + prefix) * 64, 256, device=DEV)
        plan.attend(q, kc, vc, ids, pre, out=out)
        torch.cuda.synchronize()
        assert (out == 7).all() and L.query(L.Q_KERNEL_STATUS) == 2
        plan.append(torch.ones(T, 8192, device=DEV), w, w, rot, rot, kc, vc, ids, 4096, 6144, q_out=out)
        torch.cuda.synchronize()
        assert (out == 7).all() and not kc.any() and not vc.any() and L.query(L.Q_KERNEL_STATUS) == 2


@pytest.mark.parametrize("nH,nkv,hd", [(16, 8, 256), (8, 1, 128), (4, 2, 512)])
@pytest.mark.parametrize("sign", [-1.0, 1.0])
def test_prompts_whose_scores_are_of_the_largest(nH, nkv, hd, sign):
    """As above, where rows share a tile: equal scores far from zero give equal weights, the values' running mean."""
    n = 300
    bt = Batch(nH, nkv, hd, 64, [n], [n], 0, seed=52).fill()
    bt.kc.copy_(torch.where(torch.isnan(bt.kc), bt.kc, torch.full_like(bt.kc, sign * 60000.0)))
    out = _attend(bt, torch.full_like(bt.queries(), 200.0)).view(n, nH, hd).to(F64)
    pg, sl = bt.places(0, n)
    v = bt.vc[pg, :, sl].to(F64).repeat_interleave(nH // nkv, 1)
    count = torch.arange(1, n + 1, dtype=F64, device=DEV)[:, None, None]
    mean, a = v.cumsum(0) / count, v.abs().cumsum(0) / count
    assert ((out - mean).abs() <= 2.0 ** -11 * mean.abs() + 2 * (2.0 ** -11 + 2.0 ** -20) * a + 2.0 ** -25).all()
    assert L.query(L.Q_KERNEL_STATUS) == 0


@pytest.mark.parametrize("nH,nkv,hd", [(16, 8, 256), (8, 1, 128), (4, 2, 512)])
@pytest.mark.parametrize("step", [1, 2, 3])
def test_large_scores_that_grow(nH, nkv, hd, step):
    """Scores of 2^27 to 2^28 that grow by 16 steps with every unit: all are multiples of 16, so every sum is exact in
    32 bits, and with scale log2(e) = 1 a weight of a smaller score is at most 2^-16.  Only a row's largest count."""
    n, scale = 600, float(np.float32(np.log(2)))
    assert np.float32(scale) * np.float32(1.4426950408889634) == 1
    bt = Batch(nH, nkv, hd, 64, [n], [n], 0, seed=53).fill()
    pg, sl = bt.places(0, n)
    grown = 16.0 * step * (torch.arange(n, device=DEV) // 64)
    q = torch.full_like(bt.queries(), 512.0)
    big = 156_000_000 // (512 * (hd - 1)) // 8 * 8           # f16 holds multiples of 8 up to 2^14
    q.view(n, nH, hd)[:, :, 0] = 1.0
    bt.kc[pg, :, sl] = float(big)
    bt.kc[pg, :, sl, 0] = grown.half()[:, None]
    assert 2 ** 27 <= 512 * (hd - 1) * big and 512 * (hd - 1) * big + 1000 < 2 ** 28
    out = _attend(bt, q, scale=scale).view(n, nH, hd).to(F64)
    s = torch.where(torch.tril(torch.ones(n, n, dtype=torch.bool, device=DEV)), grown.to(F64), -torch.inf)
    p = torch.exp2(s - s.amax(1, keepdim=True))
    p /= p.sum(1, keepdim=True)
    v = bt.vc[pg, :, sl].to(F64).repeat_interleave(nH // nkv, 1)
    ref, a = torch.einsum("ij,jhd->ihd", p, v), torch.einsum("ij,jhd->ihd", p, v.abs())
    assert ((out - ref).abs() <= 2.0 ** -11 * ref.abs() + 2 * (2.0 ** -11 + 2.0 ** -20) * a + 2.0 ** -25).all()
    assert L.query(L.Q_KERNEL_STATUS) == 0


RUNS = [([600, 90], [600, 300], 0, 0),                            # prompts
        ([200, 70], [900, 800], 300, 257),                        # chunks under a window
        ([1] * 70, [801 + i for i in range(70)], 800, 0),         # many users of a prefix
        ([1, 3, 2], [500, 700, 60], 40, 0)]                       # and a few rows by themselves


def _whole_scores(bt, n):
    """Keys, and queries, of -1, 0 and 1: scores are whole numbers, exact in any order."""
    ints = lambda *s: torch.randint(-1, 2, s, generator=bt.g, device=DEV).half()  # noqa: E731
    bt.kc.copy_(torch.where(torch.isnan(bt.kc), bt.kc, ints(*bt.kc.shape)))
    return ints(bt.T, n)


@pytest.mark.parametrize("nH,nkv,hd", [(16, 8, 256), (8, 1, 128), (4, 2, 512), (16, 1, 512)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("new,total,prefix,window", RUNS)
def test_an_f32_result_has_weights_of_more_bits_than_f16(nH, nkv, hd, dtype, new, total, prefix, window):
    """With exact scores the error of the weights and of the sums is left, whichever kernel a row gets.  On a weight p_j:
    its f16 (2^-11, for an f16 result) or its two f16 parts (2^-22), 2^-29 of the row's largest where a part is below f16's
    normal range, the exponential (2^-22), the slope's two roundings over the distance to the maximum (2^-23 of it, in
    powers of two).  On the sums: at most one truncation (2^-22) of the running sum for every eight keys (two products each
    of 16), rescaling and joining (2^-20)."""
    bt = Batch(nH, nkv, hd, 32, new, total, prefix, window, seed=54).fill()
    q, scale = _whole_scores(bt, nH * hd), 0.25
    out = _attend(bt, q, out_dtype=dtype, scale=scale).view(bt.T, nH, hd).to(F64)
    half, bits = torch.finfo(dtype).eps / 2, 2.0 ** (-22 if dtype == torch.float32 else -11)
    for b in range(bt.B):
        n, t0, G = new[b], int(bt.start[b]), nH // nkv
        pg, sl = bt.places(b, total[b])
        k, v = (c[pg, :, sl].to(F64).repeat_interleave(G, 1) for c in (bt.kc, bt.vc))
        pos, j = torch.arange(total[b] - n, total[b], device=DEV)[:, None], torch.arange(total[b], device=DEV)
        see = (j <= pos) & (j > pos - window) if window else j <= pos
        s = torch.einsum("mhd,jhd->mhj", q[t0:t0 + n].to(F64).view(n, nH, hd), k) * scale
        s = torch.where(see[:, None], s, torch.full_like(s, -torch.inf))
        far = (s.amax(-1, keepdim=True) - s) * 1.4427
        p = torch.softmax(s, -1)
        dp = torch.where(see[:, None], p * (bits + 2.0 ** -22 + 2.0 ** -23 * far) + 2.0 ** -29, torch.zeros_like(p))
        ref, a = torch.einsum("mhj,jhd->mhd", p, v), torch.einsum("mhj,jhd->mhd", p, v.abs())
        lim = 2 * torch.einsum("mhj,jhd->mhd", dp, v.abs()) + a * (see.sum(1)[:, None, None] / 8 * 2.0 ** -22 + 2.0 ** -20)
        err = (out[t0:t0 + n] - ref).abs()
        lim = lim + half * ref.abs() + 2.0 ** -25
        assert (err <= lim).all(), f"{(err / lim).max().item():.2f} of the tolerance"
    assert L.query(L.Q_KERNEL_STATUS) == 0


@pytest.mark.parametrize("nH,nkv,hd", [(16, 8, 256), (8, 1, 128), (4, 2, 512), (16, 1, 512)])
@pytest.mark.parametrize("new,total,prefix,window", RUNS)
def test_equal_values_come_out_as_they_are(nH, nkv, hd, new, total, prefix, window):
    """A row divides by the sum of the weights that its products had: where all values are the same, their roundings
    cancel.  What is left, under 2^-15 by the sums' part of the bound above, is less than half a step of f16."""
    bt = Batch(nH, nkv, hd, 32, new, total, prefix, window, seed=55).fill()
    q, value = _whole_scores(bt, nH * hd), bt.randn(nkv, hd).half()
    bt.vc.copy_(torch.where(torch.isnan(bt.vc), bt.vc, value[:, None]))
    out = _attend(bt, q, scale=0.25).view(bt.T, nkv, nH // nkv, hd)
    assert torch.equal(out, value[None, :, None].expand_as(out))


@pytest.mark.parametrize("nH,nkv,hd,new", [(16, 8, 256, 1), (8, 1, 128, 2), (4, 2, 512, 3), (16, 1, 512, 1), (8, 1, 128, 20)])
@pytest.mark.parametrize("prefix", [0, 100_000])
def test_many_small_weights_add_up(nH, nkv, hd, new, prefix):
    """One key 26 powers of two above 131,071 others: each of them weighs nothing beside it, together they are 2^-9.  All
    weights are powers of two and every sum is exact, so only the result's rounding and the division are left."""
    n, scale = 1 << 17, float(np.float32(np.log(2)))
    bt = Batch(nH, nkv, hd, 1024, [new], [n + new - 1], prefix, seed=56)
    for c in (bt.kc, bt.vc):
        c.zero_()
    pg, sl = bt.place(0, 70_000)
    bt.kc[pg, :, sl, 0] = 26.0
    bt.vc.fill_(1.0)
    bt.vc[pg, :, sl] = 0.0
    q = torch.zeros(bt.T, nH * hd, dtype=torch.float16, device=DEV)
    q.view(bt.T, nH, hd)[:, :, 0] = 1.0
    out = _attend(bt, q, out_dtype=torch.float32, scale=scale).view(new, -1).to(F64)
    rest = (torch.arange(new, device=DEV)[:, None] + n - 1) * 2.0 ** -26
    assert ((out - rest / (1 + rest)).abs() <= 2.0 ** -20 * rest).all()
    assert L.query(L.Q_KERNEL_STATUS) == 0


def _append_case(nH, nkv, hd, dtype, page, new, total, prefix, keqv, seed):
    bt = Batch(nH, nkv, hd, page, new, total, prefix, seed=seed, front=1, back=2)
    nq, nk = nH * hd, nkv * hd
    koff, voff = nq, nq if keqv else nq + nk
    qkv = (bt.randn(bt.T, nq + 2 * nk + 16) * torch.exp(bt.randn(bt.T, 1))).to(dtype)[:, :-16]
    qnw, knw = 1 + 0.2 * bt.randn(hd), 1 + 0.2 * bt.randn(hd)
    n_pos = (bt.own_pages + bt.pre_pages) * page
    inv = 10000.0 ** (-torch.arange(0, hd, 2, device=DEV, dtype=F64) / hd)
    ang = torch.arange(n_pos, device=DEV, dtype=F64)[:, None] * torch.cat((inv, inv))
    return bt, (qkv, qnw, knw, ang.cos().float(), ang.sin().float()), koff, voff


@pytest.mark.parametrize("nH,nkv,hd,new", [
    (16, 8, 256, [600, 0, 5, 700]), (16, 8, 256, [300, 7, 204]), (16, 8, 256, [300, 7, 203]),   # on either side of the rule
    (16, 1, 512, [500, 1, 90]), (8, 8, 128, [1400, 2, 300]), (16, 2, 128, [900, 800, 30]),
    (8, 1, 128, [4000, 90]), (4, 2, 512, [900, 300]), (16, 8, 512, [200, 150])])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("prefix,keqv", [(0, False), (40, True)])
def test_append_of_long_prompts(nH, nkv, hd, new, dtype, prefix, keqv):
    """Batches that go to the kernel whose rows stream through shared memory, and their neighbours that do not."""
    rng = np.random.default_rng(hd)
    total = [prefix + int(rng.integers(0, 90)) + n for n in new]
    total[0] = max(new[0], prefix - 20 + new[0])              # its first tokens lie inside the prefix
    bt, args, koff, voff = _append_case(nH, nkv, hd, dtype, 32, new, total, prefix, keqv, seed=60)
    q_out = torch.full((bt.T, nH * hd), 7.0, dtype=torch.float16, device=DEV)
    bt.plan().append(*args, bt.kc, bt.vc, bt.table, koff, voff, q_out=q_out)
    torch.cuda.synchronize()
    (q, qm), (k, km), (v, vm), pos = _append_reference(bt, *args, koff, voff)
    lo, hi = int(bt.start[0]), int(bt.start[-1])
    _close16(q_out.view(bt.T, nH, hd)[lo:hi], q[lo:hi], qm[lo:hi], "q")
    assert (q_out[:lo] == 7).all() and (q_out[hi:] == 7).all()
    written = torch.zeros(bt.pages, 32, dtype=torch.bool, device=DEV)
    for b in range(bt.B):
        t0, n = int(bt.start[b]), new[b]
        pg, sl = bt.places(b, total[b])
        at = torch.arange(total[b] - n, total[b], device=DEV)
        own = at >= prefix
        pg, sl, t = pg[at[own]], sl[at[own]], torch.arange(t0, t0 + n, device=DEV)[own]
        written[pg, sl] = True
        _close16(bt.kc[pg, :, sl], k[t], km[t], "k")
        _close16(bt.vc[pg, :, sl], v[t], vm[t], "v")
    for c in (bt.kc, bt.vc):
        assert torch.isnan(c.permute(0, 2, 1, 3)[~written]).all()
    assert L.query(L.Q_KERNEL_STATUS) == 0


def test_two_threads_with_long_prompts_of_other_sizes():
    """Two host threads whose appends stream through different amounts of shared memory."""
    import threading

    cases = [_append_case(16, 8, 256, torch.float16, 32, [700], [700], 0, False, 61),
             _append_case(16, 1, 512, torch.float32, 32, [500, 40], [500, 40], 0, False, 62)]
    jobs, errors = [], []
    for bt, args, koff, voff in cases:
        plan, out = bt.plan(), torch.empty(bt.T, bt.nH * bt.hd, dtype=torch.float16, device=DEV)
        jobs.append((bt, plan, (*args, bt.kc, bt.vc, bt.table, koff, voff, out), torch.cuda.Stream()))
    torch.cuda.synchronize()

    def run(bt, plan, args, stream):
        try:
            for _ in range(100):
                plan.append(*args, stream=stream)
        except Exception as e:                               # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=run, args=j) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors and L.query(L.Q_KERNEL_STATUS) == 0
    for bt, _, args, _ in jobs:
        (q, qm), (k, km), _, _ = _append_reference(bt, *args[:5], args[8], args[9])
        lo, hi = int(bt.start[0]), int(bt.start[-1])
        _close16(args[10].view(bt.T, bt.nH, bt.hd)[lo:hi], q[lo:hi], qm[lo:hi], "q")
        pg, sl = bt.places(0, bt.total[0])
        _close16(bt.kc[pg, :, sl], k[1:1 + bt.total[0]], km[1:1 + bt.total[0]], "k")


@pytest.mark.parametrize("nH,nkv,hd,new", [(16, 8, 256, 70), (16, 1, 512, 20), (4, 2, 512, 90), (8, 1, 128, 40)])
@pytest.mark.parametrize("prefix", [0, 50])
def test_values_out_of_sight_do_not_reach_an_f32_row(nH, nkv, hd, new, prefix):
    """A value that is not finite where only a tile's first token sees it, and one that only its last token sees."""
    window = 20
    bt = Batch(nH, nkv, hd, 16, [new, 1], [new + 60, 90], prefix, window, seed=63).fill()
    q = bt.queries()
    clean = _attend(bt, q, out_dtype=torch.float32)
    bt.check(clean, q)
    for p, value in ((60 - window + 1, float("nan")), (new + 59, float("inf"))):
        pg, sl = bt.place(0, p)
        bt.kc[pg, :, sl], bt.vc[pg, :, sl] = float("inf"), value
    out = _attend(bt, q, out_dtype=torch.float32)
    blind = [i for i in range(bt.T) if i not in (0, new - 1)]
    assert torch.equal(out[blind], clean[blind]) and not torch.isfinite(out[[0, new - 1]]).any()


@pytest.mark.parametrize("nH,nkv,hd", [(16, 8, 256), (8, 1, 128), (4, 2, 512)])
def test_an_infinity_leaves_the_rows_that_do_not_see_it_exact(nH, nkv, hd):
    """The last token's value is infinite, which only its own row sees: f32 rows of the same tile are as exact as elsewhere."""
    n = 100
    bt = Batch(nH, nkv, hd, 32, [n], [n], 0, seed=64).fill()
    q = _whole_scores(bt, nH * hd)
    pg, sl = bt.place(0, n - 1)
    bt.vc[pg, :, sl] = float("inf")
    out = _attend(bt, q, out_dtype=torch.float32, scale=0.25).view(n, nH, hd).to(F64)
    pg, sl = bt.places(0, n)
    k, v = (c[pg, :, sl].to(F64).repeat_interleave(nH // nkv, 1) for c in (bt.kc, bt.vc))
    see = torch.tril(torch.ones(n, n, dtype=torch.bool, device=DEV))[:-1, :-1]
    s = torch.einsum("mhd,jhd->mhj", q.to(F64).view(n, nH, hd), k)[:-1, :, :-1] * 0.25
    p = torch.softmax(torch.where(see[:, None], s, -torch.inf), -1)
    ref, a = (torch.einsum("mhj,jhd->mhd", p, x[:-1]) for x in (v, v.abs()))
    # weights 2^-21 and the slope over a distance of at most 2^7 steps (2^-16), sums 2^-18
    assert ((out[:-1] - ref).abs() <= 2.0 ** -15 * a + 2.0 ** -29 * v[:-1].abs().sum(0)).all()
    assert not torch.isfinite(out[-1]).any()


@pytest.mark.parametrize("nH,nkv,hd", [(16, 8, 256), (8, 1, 128), (4, 2, 512)])
def test_f32_results_at_scores_of_the_largest(nH, nkv, hd):
    n = 300
    bt = Batch(nH, nkv, hd, 64, [n], [n], 0, seed=65).fill()
    bt.kc.copy_(torch.where(torch.isnan(bt.kc), bt.kc, torch.full_like(bt.kc, -60000.0)))
    out = _attend(bt, torch.full_like(bt.queries(), 200.0), out_dtype=torch.float32).view(n, nH, hd).to(F64)
    pg, sl = bt.places(0, n)
    v = bt.vc[pg, :, sl].to(F64).repeat_interleave(nH // nkv, 1)
    count = torch.arange(1, n + 1, dtype=F64, device=DEV)[:, None, None]
    # equal weights, each a power of two: n / 8 truncations of the running sums are left
    assert ((out - v.cumsum(0) / count).abs() <= (n / 8 * 2.0 ** -22 + 2.0 ** -20) * v.abs().cumsum(0) / count + 2.0 ** -25).all()
