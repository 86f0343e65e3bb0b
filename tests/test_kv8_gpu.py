"""The 8-bit cache's kernels against the 64-bit restatement
(oracle/kv8_oracle.py), through the C ABI.

store and load have to be right bit for bit: 127 x is exact in fp32, a quotient
of two bf16 numbers is either a half or at least 2^-16 of itself from one, scale = top / 127
and q * scale are one fp32 operation each and the result is rounded to bf16 once.

Attention: the cache after the call is what the oracle attends over, so a new
key on a rounding border does not matter; how well it was rounded is checked
by itself.  An output may be off by
  2^-8 |ref|  its rounding to bf16, and relative to mag = sum |p v| / sum p:
  2^-11       w = p * v_scale in fp16,
  2 d         the scores, d = reach * (2 D + 64) * 2^-24 * 2: each of at most 2 D fp32
              additions and about 64 operations of the norm, the rotation, the
              scales and the exponent's argument, relative to reach = max sum |q k| *
              sm_scale; twice, for p and for the sum of p;
  2 * 2^-20 grid  q's 21 bits: each channel is off by half a step of 2^(e - 20) with
              2^e <= 2 max|q|, so a score by 2^-20 of grid = max|q| * max sum |k| * sm_scale;
  (n + 64) 2^-22  the sums over n slots, exponentials and rescaling factors in fp32;
and, fp16 having no steps below 2^-24, by 2^-25 of the unit for each of n slots times
|v| <= 128, the unit being at most 2^-14 of the largest w: 2^-39 step.
A new key before its rounding may be off by (D + 64) 2^-24 of the row's
largest (norm and rotation in fp32), so |q - 127 k / top| <= 0.5 + 127 * 4 * (D
+ 64) * 2^-24: 0.506."""

import ctypes
import math
import random

import pytest
import torch

from oracle import kv8_oracle as ko
from qdec import capi

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
EPS = 1e-6
BF = torch.bfloat16
NAN = math.nan


@pytest.fixture(scope="module")
def lib(qlib):
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return qlib


def stream():
    return torch.cuda.current_stream().cuda_stream


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32)


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def cache(g, B, nkv, cap, D):
    """A cache of random bytes, -128 among them, with scales."""
    c = {"k8": torch.randint(-128, 128, (B, nkv, cap, D), generator=g, device=DEV, dtype=torch.int8),
         "v8": torch.randint(-128, 128, (B, nkv, cap // 16, D, 16), generator=g, device=DEV, dtype=torch.int8)}
    c["k_scale"] = torch.rand((B, nkv, cap), generator=g, device=DEV) * 0.02 + 0.001
    c["v_scale"] = torch.exp(2 * randn(g, B, nkv, cap)) * 0.02
    return c


def ptrs(c):
    return {k: c[k].data_ptr() for k in ("k8", "v8", "k_scale", "v_scale")}


def slab(rows, cap, fill=NAN):
    """Rows [B, nkv, n, D] as a (K, V) slab pair of cap slots, `fill` behind."""
    B, h, n, D = rows[0].shape
    pad = torch.full((B, h, cap - n, D), fill, device=DEV, dtype=BF)
    k, v = (torch.cat([x.to(BF), pad], 2) for x in rows)
    return k, v.view(B, h, cap // 8, 8, D).transpose(3, 4).contiguous()


# ------------------------------------------------------------------ store, load

SHAPES = [(1, 1, 64, 0, 1), (2, 3, 128, 5, 1), (1, 8, 128, 0, 16), (3, 2, 64, 15, 2), (2, 2, 128, 16, 64), (1, 5, 64, 31, 33),
          (2, 8, 128, 100, 157), (1, 1, 128, 7, 500), (5, 3, 64, 64, 448), (2, 4, 128, 511, 1)]


def special_rows(x, rnd):
    """Rows with ties, extremes, zeros, and numbers that are not finite."""
    B, h, n, D = x.shape
    kinds = [lambda r: r.zero_(), lambda r: r.mul_(2.0 ** -110), lambda r: r.mul_(2.0 ** 100), lambda r: r.mul_(2.0 ** -90),
             lambda r: r[rnd.randrange(D)].fill_(math.inf), lambda r: r[rnd.randrange(D)].fill_(-math.inf),
             lambda r: r[rnd.randrange(D)].fill_(NAN), lambda r: r.fill_(-3.0),
             lambda r: r.copy_((torch.arange(D, device=DEV) % 9 - 4.0) / 2),
             lambda r: r.copy_(torch.where(torch.arange(D, device=DEV) % 2 == 0, 1.0, 0.5)),
             lambda r: r.copy_(torch.where(torch.arange(D, device=DEV) == 3, 254.0, (torch.arange(D, device=DEV) % 7).float())),
             lambda r: r.fill_(torch.finfo(BF).max), lambda r: r.fill_(2.0 ** -100)]
    for i in range(min(4 * len(kinds), B * h * n)):
        kinds[i % len(kinds)](x[rnd.randrange(B), rnd.randrange(h), rnd.randrange(n)])
    return x


@pytest.mark.parametrize("B,nkv,D,pos,n", SHAPES)
def test_store(lib, B, nkv, D, pos, n):
    g, rnd = gen(pos + n), random.Random(n)
    cap = (pos + n + 63) // 64 * 64 + 64
    slab_cap = (pos + n + 31) // 32 * 32
    src = [special_rows((randn(g, B, nkv, pos + n, D) * torch.exp(randn(g, B, nkv, pos + n, 1))).to(BF), rnd) for _ in range(2)]
    ks, vs = slab(src, slab_cap)
    c = cache(g, B, nkv, cap, D)
    before = {k: v.clone() for k, v in c.items()}
    lib.kv8_store(capi.Kv8StoreArgs(k_slab=ks.data_ptr(), v_slab=vs.data_ptr(), batch=B, nkv=nkv, head_dim=D, cap=cap,
                                    slab_cap=slab_cap, pos0=pos, n=n, **ptrs(c)), stream())
    rows = slice(pos, pos + n)
    for q8, sc, x, was8, was in ((c["k8"], c["k_scale"], src[0], before["k8"], before["k_scale"]),
                                 (ko.row_major(c["v8"]), c["v_scale"], src[1], ko.row_major(before["v8"]), before["v_scale"])):
        q, s = ko.hold(x[:, :, rows])
        bad = (q8[:, :, rows].double() != q).nonzero().tolist()
        assert not bad, f"{len(bad)} values differ, the first at {bad[0]}"
        torch.testing.assert_close(sc[:, :, rows], s.float(), rtol=0, atol=0, equal_nan=True)
        keep = torch.ones(cap, dtype=torch.bool, device=DEV)
        keep[rows] = False
        assert torch.equal(q8[:, :, keep], was8[:, :, keep]) and torch.equal(sc[:, :, keep], was[:, :, keep])


@pytest.mark.parametrize("B,nkv,D,pos,n", SHAPES)
@pytest.mark.parametrize("where", ["ragged", "none", "outside"])
def test_load(lib, B, nkv, D, pos, n, where):
    g, rnd = gen(pos + n), random.Random(n)
    cap = (pos + n + 63) // 64 * 64 + 64
    slab_cap = (n + 31) // 32 * 32 + 32
    c = cache(g, B, nkv, cap, D)
    c["k_scale"][:, :, pos], c["v_scale"][:, :, pos] = NAN, 0.0
    starts = {"ragged": [rnd.randint(0, cap - n) for _ in range(B)], "none": [0] * B,
              "outside": [rnd.choice([-2 ** 31, -n, -3, cap - n + 5, cap, 2 ** 31 - 1, 2 ** 31 - n]) for _ in range(B)]}[where]
    st = i32(starts)
    ks, vs = (torch.full((B, nkv, slab_cap, D), 7.0, dtype=BF, device=DEV),
              torch.full((B, nkv, slab_cap // 8, D, 8), 7.0, dtype=BF, device=DEV))
    lib.kv8_load(capi.Kv8LoadArgs(starts=None if where == "none" else st.data_ptr(), k_slab=ks.data_ptr(), v_slab=vs.data_ptr(),
                                  batch=B, nkv=nkv, head_dim=D, cap=cap, slab_cap=slab_cap, n=n, **ptrs(c)), stream())
    for got, q8, sc in ((ks, c["k8"], c["k_scale"]), (ko.slab_rows(vs), ko.row_major(c["v8"]), c["v_scale"])):
        assert bool((got[:, :, n:] == 7.0).all())
        full = (q8.float() * sc[..., None]).to(BF)
        for b, s in enumerate(starts):
            want = torch.full((nkv, n, D), NAN, dtype=BF, device=DEV)
            lo, hi = max(0, s), min(cap, s + n)
            if lo < hi:
                want[:, lo - s:hi - s] = full[b, :, lo:hi]
            torch.testing.assert_close(got[b, :, :n], want, rtol=0, atol=0, equal_nan=True)


# ------------------------------------------------------------------- attention


class Call:
    """One attention call on random inputs; ``run()`` leaves out and the cache."""

    def __init__(self, lib, B, nq, nkv, D, T, lens, cap=None, splits=0, frag=0, seed=1, gain=1.0):
        g = gen(seed)
        self.lib, self.B, self.nq, self.nkv, self.D, self.T, self.lens = lib, B, nq, nkv, D, T, list(lens)
        self.cap = cap or (max(lens) + T + 63) // 64 * 64
        self.c = cache(g, B, nkv, self.cap, D)
        for b, L in enumerate(lens):  # an earlier request's slots
            self.c["k_scale"][b, :, max(L, 0)::2] = NAN
            self.c["v_scale"][b, :, max(L, 0)::3] = NAN
            self.c["v_scale"][b, :, max(L, 0) + 1::3] = 3e38
        self.qkv = randn(g, B * T, (nq + 2 * nkv) * D).to(BF)
        self.qw = ((1 + 0.1 * randn(g, D)) * gain).to(BF)
        self.kw = (1 + 0.1 * randn(g, D)).to(BF)
        ang = torch.arange(self.cap)[:, None] * (1e6 ** (-torch.arange(0, D, 2) / D))[None]
        ang = torch.cat((ang, ang), -1)
        self.cos, self.sin = ang.cos().to(DEV, BF), ang.sin().to(DEV, BF)
        self.lens_t = i32(self.lens)
        rows = (B * T + 15) // 16 * 16 if frag else B * T
        self.out = torch.full((rows, nq * D), 9.0, dtype=BF, device=DEV)
        self.frag = frag
        a = self.a = capi.Kv8AttnArgs(qkv=self.qkv.data_ptr(), q_norm_w=self.qw.data_ptr(), k_norm_w=self.kw.data_ptr(),
                                      cos_tab=self.cos.data_ptr(), sin_tab=self.sin.data_ptr(), lens=self.lens_t.data_ptr(),
                                      out=self.out.data_ptr(), eps=EPS, sm_scale=D ** -0.5, batch=B, t_rows=T, nq=nq, nkv=nkv,
                                      head_dim=D, cap=self.cap, splits=splits, out_frag=frag, **ptrs(self.c))
        pb, _ = lib.kv8_attn_workspace(a)
        self.partial = torch.full((pb // 4 + 4,), NAN, device=DEV)
        a.partial = self.partial.data_ptr()

    def run(self, s=None):
        self.lib.kv8_attn(self.a, s or stream())
        return self

    def rows(self):
        """The output rows [B, T, nq, D], whatever layout they were asked in."""
        o = self.out
        if self.frag:
            nmt = o.shape[0] // 16
            o = o.view(-1).view(self.nq * self.D // 32, nmt, 4, 16, 8).permute(1, 3, 0, 2, 4).reshape(nmt * 16, -1)[:self.B * self.T]
        return o.view(self.B, self.T, self.nq, self.D)

    def check(self, before):
        B, T, nq, nkv, D = self.B, self.T, self.nq, self.nkv, self.D
        x = self.qkv.view(B, T, nq + 2 * nkv, D)
        got, vr = self.rows().double(), ko.row_major(self.c["v8"])
        for b, L in enumerate(self.lens):
            pos = slice(L, L + T)
            tab = self.cos[pos], self.sin[pos]
            # what the call wrote, and nothing else
            for q8, sc, x8, want in ((self.c["k8"], self.c["k_scale"], before["k8"],
                                      ko.norm_rope(x[b, :, nq:nq + nkv], self.kw, *tab, EPS)),
                                     (vr, self.c["v_scale"], ko.row_major(before["v8"]), x[b, :, nq + nkv:].double())):
                want = want.transpose(0, 1)
                top = want.abs().amax(-1)
                low = top < 2 ** -100  # held as zeros
                top = top.masked_fill(low, 0)
                off = (q8[b, :, pos].double() - (127 * want / top[..., None]).masked_fill(low[..., None], 0)).abs().max()
                assert off <= 0.5 + 127 * 4 * (D + 64) * 2 ** -24, f"new rows of sequence {b} off by {off} steps"
                torch.testing.assert_close(sc[b, :, pos].double(), top / 127, rtol=2 * (D + 64) * 2 ** -24, atol=0)
                keep = torch.ones(self.cap, dtype=torch.bool, device=DEV)
                keep[pos] = False
                assert torch.equal(q8[b][:, keep], x8[b][:, keep])
            q = ko.norm_rope(x[b, :, :nq], self.qw, *tab, EPS)
            ref, mag, step, reach, grid = ko.attend(q, self.c["k8"][b], self.c["k_scale"][b], self.c["v8"][b], self.c["v_scale"][b], L, D ** -0.5)
            tol = 2 ** -8 * ref.abs() + mag * (2 ** -11 + 4 * reach * (2 * D + 64) * 2 ** -24 + 2 ** -19 * grid + (L + T + 64) * 2 ** -22)
            tol += step * 2 ** -39
            bad = ~((got[b] - ref).abs() <= tol)
            assert not bool(bad.any()), (f"sequence {b} of length {L}: {int(bad.sum())} outputs off, worst "
                                         f"{((got[b] - ref).abs() / tol).max().item():.3g} of the tolerance at "
                                         f"{bad.nonzero()[0].tolist()}")

    def checked(self):
        before = {k: v.clone() for k, v in self.c.items()}
        self.run()
        torch.cuda.synchronize()
        self.check(before)
        for k in ("k_scale", "v_scale"):
            for b, L in enumerate(self.lens):
                keep = torch.ones(self.cap, dtype=torch.bool, device=DEV)
                keep[L:L + self.T] = False
                torch.testing.assert_close(self.c[k][b][:, keep], before[k][b][:, keep], rtol=0, atol=0, equal_nan=True)
        return self


# batch, nq, nkv, D, T, lengths
ATTN = [
    (1, 8, 2, 64, 1, [0]), (1, 32, 8, 128, 1, [0]), (1, 1, 1, 64, 1, [1]), (2, 4, 4, 128, 2, [63, 0]),
    (3, 32, 8, 128, 1, [63, 64, 65]), (3, 8, 2, 64, 3, [61, 62, 127]), (1, 32, 8, 128, 9, [640]), (1, 32, 8, 128, 16, [503]),
    (2, 40, 8, 128, 3, [700, 129]), (2, 64, 8, 128, 8, [300, 60]), (1, 16, 8, 128, 16, [1000]), (4, 16, 8, 128, 4, [0, 2001, 511, 512]),
    (1, 16, 1, 64, 4, [200]), (1, 64, 1, 128, 1, [333]), (2, 9, 3, 64, 5, [575, 576]), (8, 32, 8, 128, 1, [900, 1535, 1, 0, 1023, 1024, 1025, 77]),
    (5, 32, 8, 128, 2, [4100, 50, 3000, 64, 4095]), (1, 64, 8, 128, 1, [20011]), (1, 8, 2, 64, 10, [5837]),
    # several row tiles, workgroups in no whole eights; new rows on either side of a run's end
    (3, 12, 3, 64, 16, [500, 1020, 0]), (1, 20, 5, 128, 16, [1017]), (7, 64, 1, 64, 1, [511, 512, 513, 1023, 1024, 1535, 1536]),
    # one split of runs of 256 slots
    (33, 32, 8, 128, 1, [97 * i % 700 for i in range(33)]), (9, 16, 8, 128, 6, [63 * i for i in range(9)]), (65, 8, 4, 64, 3, [11 * i for i in range(65)]),
    # splits that share a workgroup, runs of 512 slots and of 256
    (4, 32, 8, 128, 9, [1100, 255, 768, 1143]), (3, 48, 6, 64, 8, [2040, 256, 1023]),
    (5, 64, 8, 128, 8, [2600, 511, 0, 1537, 2048]), (11, 24, 4, 64, 10, [3000, 90, 1024, 1526, 600, 5, 1018, 2999, 64, 512, 1800]),
    (1, 32, 8, 128, 16, [1531]), (2, 8, 8, 128, 16, [507, 2045]), (3, 7, 7, 128, 1, [63, 64, 512]), (2, 48, 4, 128, 5, [2100, 3]),
]


@pytest.mark.parametrize("shape", ATTN, ids=[f"{s[0]}x{s[1]}/{s[2]}x{s[3]}-t{s[4]}-{max(s[5])}" for s in ATTN])
def test_attention(lib, shape):
    Call(lib, *shape).checked()


@pytest.mark.parametrize("splits", [1, 2, 3, 7, 64])
@pytest.mark.parametrize("T", [1, 5])
def test_splits(lib, splits, T):
    Call(lib, 3, 32, 8, 128, T, [1500, 130, 0], splits=splits).checked()
    Call(lib, 2, 8, 2, 64, T, [60, 900], splits=splits, seed=2).checked()


@pytest.mark.parametrize("shape", [(3, 32, 8, 128, 4, [100, 3, 700]), (17, 8, 2, 64, 1, [5 * b for b in range(17)])])
@pytest.mark.parametrize("splits", [1, 3])
def test_fragment_order(lib, shape, splits):
    a = Call(lib, *shape, splits=splits, frag=1).checked()
    b = Call(lib, *shape, splits=splits).run()
    assert torch.equal(a.rows(), b.rows())


@pytest.mark.parametrize("shape", [(3, 12, 3, 64, 16, [500, 1020, 505]), (1, 64, 8, 128, 8, [1533]), (1, 32, 8, 128, 16, [2040])])
@pytest.mark.parametrize("splits", [2, 3])
def test_new_rows_in_two_splits(lib, shape, splits):
    Call(lib, *shape, splits=splits).checked()


@pytest.mark.parametrize("q,k", [(1e30, 1e-28), (1e-28, 1e30), (3e36, 1e-34), (1e-20, 1e-20)])
def test_norm_gains_of_any_size(lib, q, k):
    """Queries and new keys far from 1, among cached keys as far from it."""
    a = Call(lib, 1, 32, 8, 128, 2, [300])
    a.qw.mul_(q), a.kw.mul_(k)
    a.c["k_scale"].mul_(k)
    a.checked()


@pytest.mark.parametrize("gain", [0.01, 30.0])
def test_flat_and_peaked_scores(lib, gain):
    Call(lib, 2, 32, 8, 128, 3, [1200, 70], gain=gain).checked()


@pytest.mark.parametrize("shape", [(2, 32, 8, 128, [700, 61]), (1, 64, 8, 128, [1022]), (3, 8, 2, 64, [0, 63, 500]),
                                   (2, 16, 8, 128, [509, 1021]), (1, 30, 3, 64, [1533]),
                                   (5, 64, 8, 128, [1500, 1021, 3, 1533, 700]), (4, 64, 8, 128, [1100, 253, 766, 1]),
                                   (33, 32, 8, 128, [53 * i for i in range(33)]), (9, 40, 8, 128, [55 * i for i in range(9)])])
@pytest.mark.parametrize("splits", [0, 1, 3])
def test_rows_do_not_depend_on_the_pass(lib, shape, splits):
    """One pass of 6 rows and 6 passes of one leave the same bits, in the rows
    and in the cache."""
    B, nq, nkv, D, lens = shape
    T, cap = 6, (max(lens) + 6 + 63) // 64 * 64
    whole = Call(lib, B, nq, nkv, D, T, lens, cap=cap, splits=splits)
    start = {k: v.clone() for k, v in whole.c.items()}
    whole.run()
    one = Call(lib, B, nq, nkv, D, 1, lens, cap=cap, splits=splits)
    for k, v in start.items():
        one.c[k].copy_(v)
    one.qw.copy_(whole.qw), one.kw.copy_(whole.kw)
    x = whole.qkv.view(B, T, -1)
    for t in range(T):
        one.qkv.copy_(x[:, t])
        one.lens_t.copy_(i32([L + t for L in lens]))
        one.run()
        assert torch.equal(one.rows()[:, 0], whole.rows()[:, t]), f"row {t}"
    for k in start:
        torch.testing.assert_close(one.c[k], whole.c[k], rtol=0, atol=0, equal_nan=True)


def test_sequences_do_not_depend_on_each_other(lib):
    a = Call(lib, 3, 32, 8, 128, 2, [900, 64, 300], cap=1024).run()
    b = Call(lib, 3, 32, 8, 128, 2, [900, 64, 300], cap=1024)
    b.lens_t.copy_(i32([0, 64, 1000]))
    for k in ("k_scale", "v_scale"):
        b.c[k][0], b.c[k][2] = NAN, NAN
    b.run()
    assert torch.equal(a.rows()[1], b.rows()[1])


@pytest.mark.parametrize("bad", [-1, -2 ** 31, 127, 1 << 20, 2 ** 31 - 1])
@pytest.mark.parametrize("splits", [1, 2])
def test_invalid_length(lib, bad, splits):
    """Length bad of cap 128 with 2 rows: NaN rows, no cache memory touched."""
    a = Call(lib, 2, 8, 2, 64, 2, [40, 70], cap=128, splits=splits)
    a.lens_t.copy_(i32([40, bad]))
    before = {k: v.clone() for k, v in a.c.items()}
    a.run()
    assert bool(torch.isnan(a.rows()[1]).all()) and not bool(torch.isnan(a.rows()[0]).any())
    for k in before:
        torch.testing.assert_close(a.c[k][1], before[k][1], rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("splits", [1, 4])
@pytest.mark.parametrize("T", [1, 3])
def test_values_of_many_magnitudes(lib, splits, T):
    """A value row of 1e30 or 1e-25 among ordinary ones: behind a score that
    leaves it no probability it must not cost the others their bits, with
    probability it must come out itself; zero values give zero."""
    for kind in ("hidden", "seen", "small", "zero", "last"):
        a = Call(lib, 1, 32, 8, 128, T, [900], splits=splits)
        if kind == "hidden":
            # keys opposite to every query are impossible at once; a row of queries along
            # channel 0 and one loud key against it
            x = a.qkv.view(T, -1, 128)
            x[:, :32] = 0.0
            x[:, :32, 64 - 1] = 1.0
            a.qw[63] = 16.0
            a.cos[:], a.sin[:] = 1.0, 0.0
            a.c["k8"][:, :, :, 63] = a.c["k8"][:, :, :, 63].abs()
            a.c["k8"][0, :, 100, 63] = -127
            a.c["k_scale"][0, :, 100] = 1.0
            a.c["v_scale"][0, :, 100] = 1e28
        elif kind == "seen":
            a.c["v_scale"][0, :, 100] = 1e28
        elif kind == "small":
            a.c["v_scale"][0] *= 1e-25
        elif kind == "zero":
            a.c["v_scale"][0, :, :900] = 0.0
        else:
            a.c["v_scale"][0, :, :] = 1e-6
            a.c["v_scale"][0, :, 899] = 1e20
        a.checked()


@pytest.mark.parametrize("splits", [1, 2])
@pytest.mark.parametrize("slot", [100, 600, 899])
@pytest.mark.parametrize("loud", [0.04, 0.07, 1.0, 100.0])
def test_zero_values_with_the_probability(lib, splits, slot, loud):
    """A slot whose score is far above all others, with values of zero: before
    and behind it in its wave are slots of 2^-80 of its probability and less."""
    a = Call(lib, 1, 32, 8, 128, 2, [900], splits=splits)
    x = a.qkv.view(2, -1, 128)
    x[:, :32] = 0.0
    x[:, :32, 63] = 1.0
    a.qw[63] = 16.0
    a.cos[:], a.sin[:] = 1.0, 0.0
    a.c["k_scale"][:] = 0.002
    a.c["k8"][0, :, slot, 63] = 127
    a.c["k_scale"][0, :, slot] = loud
    a.c["v_scale"][0, :, slot] = 0.0
    x[:, 32:40, 63] = 0.0
    a.run()
    got = a.rows()
    assert bool(torch.isfinite(got).all())
    # scores are 16 times the key's channel: at most 16 * 128 * 0.002 of 901 slots, 16 * 127 * loud of one
    vals = 128 * max(1.0, float(a.c["v_scale"][0, :, :902].max()))
    assert float(got.abs().max()) <= 901 * vals * math.exp(-0.99 * 16 * (127 * loud - 128 * 0.002))


def test_not_finite_where_it_is_seen(lib):
    """A NaN scale reaches the rows and heads that see its slot, no others."""
    for which in ("k_scale", "v_scale"):
        a = Call(lib, 2, 32, 8, 128, 3, [200, 150])
        a.c[which][0, 3, 17] = NAN
        a.run()
        nan = torch.isnan(a.rows())
        assert bool(nan[0, :, 12:16].all()) and int(nan.sum()) == 3 * 4 * 128
    # a value row with an infinity, in the second of three new rows
    a = Call(lib, 1, 8, 2, 64, 3, [70])
    a.qkv.view(3, 12, 64)[1, 10, 5] = math.inf
    a.run()
    nan = torch.isnan(a.rows())
    assert not bool(nan[0, 0].any()) and bool(nan[0, 1:, :4].all()) and not bool(nan[0, 1:, 4:].any())
    assert bool(torch.isnan(a.c["v_scale"][0, 0, 71])) and int(torch.isnan(a.c["v_scale"][0, :, :73]).sum()) == 1


@pytest.mark.parametrize("B,nkv,T,lens,splits", [
    (1, 8, 1, [700], 0), (1, 8, 1, [1500], 0), (1, 8, 1, [9000], 0), (1, 8, 1, [511], 3), (1, 8, 1, [512], 3), (1, 8, 1, [40], 1),
    (2, 8, 1, [3000, 90], 0), (2, 4, 1, [1023, 2600], 5), (4, 8, 1, [1022, 0, 511, 40], 2), (1, 4, 1, [17000], 33)])
@pytest.mark.parametrize("kind", ["plain", "loud", "nan"])
def test_merge_in_the_next_gemm(lib, B, nkv, T, lens, splits, kind):
    """A product that merges the partials (weights one on the diagonal, so that it
    gives its rows) has the bits of the call that merges them itself."""
    rows = []
    k = nkv * 4 * 128
    eye = torch.eye(k, device=DEV).to(BF)
    w = torch.empty_like(eye)
    lib.pack_tiles(eye.data_ptr(), w.data_ptr(), k, k, stream())
    for partials in (0, 1):
        a = Call(lib, B, 4 * nkv, nkv, 128, T, lens, splits=splits)
        if kind == "loud":
            a.c["v_scale"].mul_(1e33)
        if kind == "nan":
            a.c["k_scale"][B - 1, 1, 7] = NAN
            a.qkv[B * T - 1, 2 * 128 + 5] = math.inf
        a.a.out_partials = partials
        pb, _ = lib.kv8_attn_workspace(a.a)
        a.partial = torch.full((pb // 4 + 4,), NAN, device=DEV)
        a.a.partial = a.partial.data_ptr()
        a.run()
        res = torch.zeros((B * T, k), dtype=BF, device=DEV)
        o = capi.GemmArgs(x=a.out.data_ptr(), w=w.data_ptr(), res=res.data_ptr(), eps=EPS, rows=B * T, n=k, k=k,
                          flags=capi.RES_OUT, ksplit=1, waves=8, tiles_per_wg=1)
        if partials:
            o.x_kv8 = ctypes.addressof(a.a)
            assert bool((a.out == 9.0).all())
        lib.gemm(o, stream())
        rows.append(res)
        if not partials and kind != "nan":
            assert torch.equal(res, a.out) and bool(torch.isfinite(res).all())
    torch.testing.assert_close(rows[1], rows[0], rtol=0, atol=0, equal_nan=True)
    if kind == "nan":
        assert bool(torch.isnan(rows[0]).any())
    # a length that the attention refuses
    a.lens_t.copy_(i32([a.cap - T + 1] + lens[1:]))
    a.run()
    res = torch.zeros((B * T, k), dtype=BF, device=DEV)
    o.res = res.data_ptr()
    lib.gemm(o, stream())
    assert bool(torch.isnan(res[:T]).all())


@pytest.mark.parametrize("shape", [(2, 32, 8, 128, 1, [1500, 300]), (4, 32, 8, 128, 9, [1100, 255, 768, 1143]), (1, 8, 2, 64, 10, [3000]),
                                   (5, 64, 8, 128, 8, [1800, 40, 511, 1000, 1543]), (3, 16, 8, 128, 4, [20, 0, 500])])
@pytest.mark.parametrize("splits", [0, 3])
def test_partials(lib, shape, splits):
    """What out_partials leaves, merged in 64 bits, against the call's own rows: both
    round once to bf16, the call's with a merge in fp32."""
    B, nq, nkv, D, T, lens = shape
    a = Call(lib, *shape, splits=splits).run()
    b = Call(lib, *shape, splits=splits)
    b.a.out_partials = 1
    R, pb = T * nq // nkv, lib.kv8_attn_workspace(b.a)[0]
    C = pb // (4 * B * nkv * R * (D + 2))
    b.partial = torch.full((pb // 4 + 4,), NAN, device=DEV)
    b.a.partial = b.partial.data_ptr()
    b.run()
    assert bool((b.out == 9.0).all()) and bool(torch.isnan(b.partial[pb // 4:]).all())
    part = b.partial[:pb // 4].view(B, nkv, C, R * (D + 2)).double()
    acc, m, l = part[..., :R * D].reshape(B, nkv, C, R, D), part[..., R * D:R * (D + 1)], part[..., R * (D + 1):]
    left = ~torch.isnan(m)  # the splits that hold slots left theirs: as many of the first for every row
    n = left.sum(2, keepdim=True)
    assert bool((left == (torch.arange(C, device=DEV)[:, None] < n)).all()) and bool((n == n[:, :1, :, :1]).all())
    top = m.masked_fill(~left, -math.inf).amax(2, keepdim=True)
    w = torch.where(left & (m > -math.inf), torch.exp2(m - top), 0.0)
    want = (torch.where(w[..., None] > 0, acc, 0.0) * w[..., None]).sum(2) / (torch.where(w > 0, l, 0.0) * w).sum(2)[..., None]
    want = want.view(B, nkv, T, nq // nkv, D).transpose(1, 2).reshape(B, T, nq, D)
    torch.testing.assert_close(a.rows().double(), want, rtol=2 ** -8, atol=float(want.abs().max()) * 2 ** -18)


class Banded:
    """A tensor's copy in the middle of a larger buffer."""

    def __init__(self, x, band=4096):
        n = x.numel() * x.element_size()
        self.buf = torch.full((n + 2 * band,), 0x5a, dtype=torch.uint8, device=DEV)
        self.t = self.buf[band:band + n].view(x.dtype).view(x.shape)
        self.t.copy_(x)
        self.band = band

    def whole(self):
        return bool((self.buf[:self.band] == 0x5a).all()) and bool((self.buf[-self.band:] == 0x5a).all())


@pytest.mark.parametrize("shape", [(2, 32, 8, 128, 1, [1087, 0]), (1, 64, 8, 128, 8, [2040]), (3, 9, 3, 64, 5, [59, 123, 0]), (5, 40, 8, 128, 1, [639] * 5)])
@pytest.mark.parametrize("splits", [0, 1, 7])
def test_guard_bands(lib, shape, splits):
    """Nothing is written outside the tensors, with the last slots of the cache taken."""
    a = Call(lib, *shape, splits=splits, frag=shape[0] * shape[4] >= 5)
    pb, _ = lib.kv8_attn_workspace(a.a)
    held = {k: Banded(v) for k, v in a.c.items()}
    out, part = Banded(a.out), Banded(torch.zeros(max(pb, 16) // 4, device=DEV))
    for k, v in held.items():
        setattr(a.a, k, v.t.data_ptr())
    a.a.out, a.a.partial = out.t.data_ptr(), part.t.data_ptr()
    a.run()
    n, slots, st = a.cap - 7, (a.cap + 31) // 32 * 32, i32([7] * a.B)
    rows = [randn(gen(4), a.B, a.nkv, a.cap, a.D).to(BF) for _ in range(2)]
    ks, vs = (Banded(x) for x in slab(rows, slots))
    both = dict(k_slab=ks.t.data_ptr(), v_slab=vs.t.data_ptr(), batch=a.B, nkv=a.nkv, head_dim=a.D, cap=a.cap, slab_cap=slots, n=n,
                **{k: v.t.data_ptr() for k, v in held.items()})
    lib.kv8_store(capi.Kv8StoreArgs(pos0=7, **both), stream())
    lib.kv8_load(capi.Kv8LoadArgs(starts=st.data_ptr(), **both), stream())
    torch.cuda.synchronize()
    assert all(x.whole() for x in (*held.values(), out, part, ks, vs))


def test_run_of_the_operators(lib):
    """A prompt's slots stored, steps over them, and a read back of all of it
    into slabs that are stored again.  A row held from bf16 numbers comes back
    the same: its largest is read back exactly and q scale is rounded by at most 127
    * 2^-8 = 0.496 steps.  A step's key was held from fp32, so its largest is
    rounded too and 127 x / top moves by at most 127 * 2 * 2^-8 < 1: one step."""
    B, nkv, D, n = 2, 8, 128, 333
    g = gen(5)
    a = Call(lib, B, 32, nkv, D, 2, [n, n], cap=384)
    rows = [randn(g, B, nkv, n, D).to(BF) for _ in range(2)]
    ks, vs = slab(rows, 352)
    lib.kv8_store(capi.Kv8StoreArgs(k_slab=ks.data_ptr(), v_slab=vs.data_ptr(), batch=B, nkv=nkv, head_dim=D, cap=384,
                                    slab_cap=352, pos0=0, n=n, **ptrs(a.c)), stream())
    a.checked()
    k2, v2 = slab([r[:, :, :0] for r in rows], 384)
    lib.kv8_load(capi.Kv8LoadArgs(k_slab=k2.data_ptr(), v_slab=v2.data_ptr(), batch=B, nkv=nkv, head_dim=D, cap=384, slab_cap=384,
                                  n=n + 2, **ptrs(a.c)), stream())
    again = {k: torch.zeros_like(v) for k, v in a.c.items()}
    lib.kv8_store(capi.Kv8StoreArgs(k_slab=k2.data_ptr(), v_slab=v2.data_ptr(), batch=B, nkv=nkv, head_dim=D, cap=384,
                                    slab_cap=384, pos0=0, n=n + 2, **ptrs(again)), stream())
    assert torch.equal(again["k8"][:, :, :n], a.c["k8"][:, :, :n])
    assert int((again["k8"][:, :, n:n + 2].int() - a.c["k8"][:, :, n:n + 2].int()).abs().max()) <= 1
    assert torch.equal(ko.row_major(again["v8"])[:, :, :n + 2], ko.row_major(a.c["v8"])[:, :, :n + 2])


def test_graph_replays_and_streams(lib):
    """Captured on a side stream, replayed with other lengths and rows between:
    every replay equals an eager call."""
    B, T = 2, 2
    a = Call(lib, B, 32, 8, 128, T, [700, 130], cap=1024, splits=3)
    eager = Call(lib, B, 32, 8, 128, T, [700, 130], cap=1024, splits=3)
    for c in (a, eager):  # the lengths move past slots that no call writes
        c.c["k_scale"].fill_(0.01), c.c["v_scale"].fill_(0.02)
    out = torch.zeros((B, 8, 32, 128), dtype=BF, device=DEV), torch.zeros((B, 8, 4, 128, 8), dtype=BF, device=DEV)
    back = capi.Kv8LoadArgs(starts=a.lens_t.data_ptr(), k_slab=out[0].data_ptr(), v_slab=out[1].data_ptr(), batch=B, nkv=8,
                            head_dim=128, cap=1024, slab_cap=32, n=T, **ptrs(a.c))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a.run()
        lib.kv8_load(back, stream())
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.run()
        lib.kv8_load(back, stream())
    for i in range(4):
        lens, x = i32([700 + 3 * i, 130 + 60 * i]), randn(gen(i), B * T, 48 * 128).to(BF)
        for c in (a, eager):
            c.lens_t.copy_(lens)
            c.qkv.copy_(x)
        graph.replay()
        eager.run()
        torch.cuda.synchronize()
        assert bool(torch.isfinite(a.out).all()) and torch.equal(a.out, eager.out)
        for b in range(B):
            L = int(lens[b])
            want = (eager.c["k8"][b, :, L:L + T].float() * eager.c["k_scale"][b, :, L:L + T, None]).to(BF)
            assert torch.equal(out[0][b, :, :T], want)


def test_offsets_past_32_bits(lib):
    """A cache of more than 2^31 elements: the last sequence's store, step and
    read back."""
    B, nkv, D, cap = 36, 8, 128, 61440
    g = gen(9)
    c = {"k8": torch.zeros((B, nkv, cap, D), dtype=torch.int8, device=DEV),
         "v8": torch.zeros((B, nkv, cap // 16, D, 16), dtype=torch.int8, device=DEV),
         "k_scale": torch.zeros((B, nkv, cap), device=DEV), "v_scale": torch.zeros((B, nkv, cap), device=DEV)}
    assert c["k8"].numel() > 2 ** 31
    n, L = 40, cap - 1
    rows = [randn(g, B, nkv, n, D).to(BF) for _ in range(2)]
    ks, vs = slab(rows, 64)
    lib.kv8_store(capi.Kv8StoreArgs(k_slab=ks.data_ptr(), v_slab=vs.data_ptr(), batch=B, nkv=nkv, head_dim=D, cap=cap,
                                    slab_cap=64, pos0=0, n=n, **ptrs(c)), stream())
    q, _ = ko.hold(rows[0][-1])
    assert torch.equal(c["k8"][-1, :, :n].double(), q)
    q, _ = ko.hold(rows[1][-1])
    assert torch.equal(ko.row_major(c["v8"][-1, :, :4])[:, :n].double(), q)
    lens = [3] * (B - 1) + [L]
    a = Call(lib, B, 8, 8, D, 1, [3] * B, cap=64)
    cos, sin = torch.ones((cap, D), dtype=BF, device=DEV), torch.zeros((cap, D), dtype=BF, device=DEV)
    a.lens_t.copy_(i32(lens))
    a.a.cos_tab, a.a.sin_tab, a.a.cap = cos.data_ptr(), sin.data_ptr(), cap
    for k, v in ptrs(c).items():
        setattr(a.a, k, v)
    pb, _ = lib.kv8_attn_workspace(a.a)
    part = torch.zeros((pb // 4 + 4,), device=DEV)
    a.a.partial = part.data_ptr()
    a.run()
    x = a.qkv.view(B, 1, 24, D)
    tab = cos[:1], sin[:1]
    qn = ko.norm_rope(x[-1, :, :8], a.qw, *tab, EPS)
    ref, mag, step, reach, grid = ko.attend(qn, c["k8"][-1], c["k_scale"][-1], c["v8"][-1], c["v_scale"][-1], L, D ** -0.5)
    tol = 2 ** -8 * ref.abs() + mag * (2 ** -11 + 4 * reach * (2 * D + 64) * 2 ** -24 + 2 ** -19 * grid + (L + 65) * 2 ** -22) + step * 2 ** -39
    assert bool(((a.rows()[-1].double() - ref).abs() <= tol).all())
    k2, v2 = torch.zeros((B, nkv, 32, D), dtype=BF, device=DEV), torch.zeros((B, nkv, 4, D, 8), dtype=BF, device=DEV)
    lib.kv8_load(capi.Kv8LoadArgs(starts=a.lens_t.data_ptr(), k_slab=k2.data_ptr(), v_slab=v2.data_ptr(), batch=B, nkv=nkv,
                                  head_dim=D, cap=cap, slab_cap=32, n=1, **ptrs(c)), stream())
    assert torch.equal(k2[-1, :, 0], (c["k8"][-1, :, L].float() * c["k_scale"][-1, :, L, None]).to(BF))
    got = ko.slab_rows(v2)[-1, :, 0]
    assert torch.equal(got, (ko.row_major(c["v8"][-1, :, -1:])[:, -1].float() * c["v_scale"][-1, :, L, None]).to(BF))
