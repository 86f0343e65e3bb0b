"""The tree-speculation kernels against the 64-bit restatement
(oracle/tree_oracle.py), through the C ABI.

Attention inputs whose normalised, rotated rows are known exactly: query and
key entries are +-1, so x * rstd is +-1 / sqrt(1 + eps); every position turns
every channel pair by a multiple of 90 degrees (cos and sin are 0 or +-1), so a
rotated entry is +-w / sqrt(1 + eps), 5e-7 off a bf16 value, and rounds to it.
So k_nodes has to equal the restatement bit for bit, and an output differs
from it by no more than 2^-8 of itself (its rounding) and, relative to mag =
sum of |p v| / sum of p:
  2^-16  the probabilities in two bf16 parts (half a step of half a step),
  2^-10  the scores' fp32 sums: 2 * 128 * 2^-24 * sum |q k| / sqrt(D), with
         that sum at most 64 (|q|, |k| are about sqrt(D): it is about 17),
  (L + T + 64) * 2^-22  the sums over the rows, the exponentials and the
         rescaling factors in fp32.
Another test has real tables and rows.
Slots from L on hold NaN; some cached slots and all nodes hold values 64 to
256 times larger, so one row too many or too few shows at any length."""

import random

import pytest
import torch

from oracle import tree_oracle
from qdec import capi

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
EPS = 1e-6
NAN = float("nan")


@pytest.fixture(scope="module")
def lib(qlib):
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return qlib


def stream():
    return torch.cuda.current_stream().cuda_stream


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def i64(x):
    return torch.tensor(x, dtype=torch.int64, device=DEV)


def tree(kind, T, rnd):
    if kind == "chain":
        return list(range(-1, T - 1))
    if kind == "star":
        return [-1] + [0] * (T - 1)
    p = [-1] + [t - 1 if rnd.random() < 0.6 else rnd.randrange(t) for t in range(1, T)]
    if kind == "holes":  # rows that hold no node, and descendants of such rows
        for t in range(1, T):
            if rnd.random() < 0.3:
                p[t] = rnd.choice([-1, -7, t, t + 1, 99, 1 << 30, -(1 << 31)])
        p[0] = rnd.choice([-1, 0, 5, -9])  # the root's entry is not read
    if kind == "short":
        live = rnd.randint(1, T)
        p[live:] = [-1] * (T - live)
    return p


def v_layout(v):
    """[.., cap, D] -> [.., cap/8, D, 8]."""
    *lead, cap, D = v.shape
    return v.view(*lead, cap // 8, 8, D).transpose(-1, -2).contiguous()


def rope(cap, D):
    inv = 1.0 / (5e6 ** (torch.arange(0, D, 2, dtype=torch.float32) / D))
    ang = torch.arange(cap, dtype=torch.float32)[:, None] * inv
    ang = torch.cat((ang, ang), 1)
    return ang.cos().to(DEV, torch.bfloat16), ang.sin().to(DEV, torch.bfloat16)


def quarter_turns(cap, D, g):
    """cos and sin of random multiples of 90 degrees per position and pair."""
    k = torch.randint(0, 4, (cap, D // 2), generator=g, device=DEV)
    k = torch.cat((k, k), 1)
    one = torch.tensor([1, 0, -1, 0], dtype=torch.bfloat16, device=DEV)
    return one[k], one[(k + 3) % 4]


def bound(out, mag, L, T):
    return out.abs() * 2.0 ** -8 + mag * (2.0 ** -16 + 2.0 ** -10 + (L + T + 64) * 2.0 ** -22)


class Attn:
    """One attention call's tensors and argument block."""

    def __init__(self, lib, lens, T, nq, nkv, D, kind="random", splits=0, out_frag=0, seed=0, cap=None):
        g = torch.Generator(device=DEV).manual_seed(seed)
        rnd = random.Random(seed)
        B = len(lens)
        cap = cap or (max(max(lens), 0) + T + 31) // 32 * 32
        self.lib, self.lens_l, self.B, self.T, self.nq, self.nkv, self.D, self.cap = lib, lens, B, T, nq, nkv, D, cap

        def normal(*shape):
            return torch.randn(shape, generator=g, device=DEV).to(torch.bfloat16)

        self.trees = [tree(kind, T, rnd) for _ in lens]
        x = torch.sign(torch.randn((B * T, nq + 2 * nkv, D), generator=g, device=DEV)).to(torch.bfloat16)
        x[x == 0] = 1
        x[:, nq + nkv:] = 64 * normal(B * T, nkv, D)
        live = torch.tensor([u is not None for p in self.trees for u in tree_oracle.ancestors(p)], device=DEV)
        x[~live] = NAN  # rows that hold no node
        self.qkv = x.view(B * T, -1)
        self.live = live
        self.qn, self.kn = normal(D), normal(D)
        self.cos, self.sin = quarter_turns(cap, D, g)
        self.k = normal(B, nkv, cap, D)
        v = normal(B, nkv, cap, D)
        for b, L in enumerate(lens):
            for s in {0, 31, 32, L // 2, L - 1}:
                if 0 <= s < L:
                    v[b, :, s] *= 256
            self.k[b, :, max(L, 0):] = NAN
            v[b, :, max(L, 0):] = NAN
        self.v_rows = v
        self.v = v_layout(v)
        self.lens, self.parents = i32(lens), i32(self.trees)
        rows = (B * T + 15) // 16 * 16
        self.out = torch.full((rows + 1, nq * D), 3.0, dtype=torch.bfloat16, device=DEV)  # a row behind the last
        self.kno = torch.full((B, nkv, T, D), 7.0, dtype=torch.bfloat16, device=DEV)
        self.vno = torch.full((B, nkv, T, D), 7.0, dtype=torch.bfloat16, device=DEV)
        a = self.a = capi.TreeAttnArgs()
        for f, t in (("qkv", self.qkv), ("q_norm_w", self.qn), ("k_norm_w", self.kn), ("cos_tab", self.cos),
                     ("sin_tab", self.sin), ("lens", self.lens), ("parents", self.parents), ("k_cache", self.k),
                     ("v_cache", self.v), ("k_nodes", self.kno), ("v_nodes", self.vno), ("out", self.out)):
            setattr(a, f, t.data_ptr())
        a.eps, a.sm_scale, a.batch, a.t_rows, a.nq, a.nkv, a.head_dim = EPS, D ** -0.5, B, T, nq, nkv, D
        a.cap, a.splits, a.out_frag = cap, splits, out_frag
        pb, cb = lib.tree_attn_workspace(a)
        self.partial = torch.full((max(pb, 4) // 4,), NAN, dtype=torch.float32, device=DEV)
        assert cb == 0
        a.partial = self.partial.data_ptr()

    def run(self):
        self.lib.tree_attn(self.a, stream())

    def rows(self):
        """out as [B, T, nq, D] rows."""
        B, T, C = self.B, self.T, self.nq * self.D
        if not self.a.out_frag:
            return self.out[:B * T].view(B, T, self.nq, self.D)
        nmt = (B * T + 15) // 16
        x = self.out[:16 * nmt].reshape(C // 32, nmt, 4, 16, 8)  # k step, M tile, 8-channel group, row, channel
        return x.permute(1, 3, 0, 2, 4).reshape(16 * nmt, C)[:B * T].view(B, T, self.nq, self.D)

    def check(self, seqs=None):
        torch.cuda.synchronize()
        assert (self.out[(self.B * self.T + 15) // 16 * 16:] == 3.0).all()
        if not self.a.out_frag:
            assert (self.out[self.B * self.T:] == 3.0).all()
        got = self.rows().double()
        for b in seqs if seqs is not None else range(self.B):
            L, T = self.lens_l[b], self.T
            ref, mag, kn, vn = tree_oracle.attention(
                self.qkv[b * T:(b + 1) * T], self.trees[b], L, self.k[b], self.v_rows[b], self.qn, self.kn, self.cos,
                self.sin, self.nq, self.nkv, EPS)
            live = self.live[b * T:(b + 1) * T]
            assert (got[b][~live] == 0).all()
            assert (self.kno[b][:, ~live] == 7).all() and (self.vno[b][:, ~live] == 7).all()
            assert torch.equal(self.kno[b][:, live].double(), kn[:, live])
            assert torch.equal(self.vno[b][:, live].double(), vn[:, live])
            bad = ~((got[b] - ref).abs() <= bound(ref, mag, L, T))
            assert not bad.any(), (b, L, int(bad.sum()), bad.nonzero()[:3].tolist(),
                                   ((got[b] - ref).abs() / mag.clamp(min=1e-30)).nan_to_num(9).max().item())


EDGES = [0, 1, 7, 31, 32, 33, 63, 64, 65, 100, 127, 129, 255, 257]


@pytest.mark.parametrize("kind", ["chain", "star", "random", "holes", "short"])
@pytest.mark.parametrize("T", [1, 2, 5, 16, 31, 32, 33, 48, 63, 64])
def test_attention_tree_shapes(lib, T, kind):
    c = Attn(lib, EDGES[:5 if T > 16 else 14], T, 8, 2, 128, kind, seed=T)
    c.run()
    c.check()


@pytest.mark.parametrize("nq,nkv,D", [(2, 2, 64), (8, 2, 64), (16, 1, 64), (7, 7, 128), (16, 8, 128), (15, 5, 128),
                                      (40, 8, 128), (64, 8, 128), (11, 1, 128), (32, 2, 128)])
@pytest.mark.parametrize("T", [1, 3, 9, 20, 64])
def test_attention_head_layouts(lib, nq, nkv, D, T):
    c = Attn(lib, [0, 45, 300], T, nq, nkv, D, "holes", seed=nq * T)
    c.run()
    c.check()


@pytest.mark.parametrize("splits", [1, 2, 3, 7, 16, 61, 256])
@pytest.mark.parametrize("T", [4, 40])
def test_attention_splits(lib, splits, T):
    c = Attn(lib, [0, 33, 129, 500, 1024, 1999], T, 8, 2, 128, "random", splits=splits, seed=splits)
    c.run()
    c.check()
    first = [t.clone() for t in (c.out, c.kno, c.vno)]
    c.run()  # the same bits every time
    torch.cuda.synchronize()
    for x, y in zip(first, (c.out, c.kno, c.vno)):
        assert torch.equal(x.view(torch.int16), y.view(torch.int16))


@pytest.mark.parametrize("B", [2, 3, 63, 64, 65, 130])
@pytest.mark.parametrize("splits", [0, 2, 5])
@pytest.mark.parametrize("T", [2, 33])
def test_attention_ragged_batches(lib, B, splits, T):
    """Splits are dealt to the sequences by their lengths: one long among short
    ones, empty ones, and lengths out of range between them."""
    rnd = random.Random(B)
    lens = [rnd.choice([0, 3, 40, 200]) for _ in range(B)]
    lens[B // 2] = 2500
    lens[-1] = 700
    c = Attn(lib, lens, T, 4, 2, 64, "short", splits=splits, seed=B)
    bad = [b for b in range(B) if b % 7 == 4 and b != B // 2]
    now = list(lens)
    for b in bad:
        now[b] = rnd.choice([-1, 1 << 30])
    c.lens.copy_(i32(now))
    c.run()
    c.check([b for b in sorted({0, 1, B // 2 - 1, B // 2, B // 2 + 1, B - 2, B - 1}) if 0 <= b < B and b not in bad])
    for b in bad:
        assert c.rows()[b].isnan().all() and (c.kno[b] == 7).all()
    for b in range(B):
        assert b in bad or c.rows()[b].isfinite().all()


@pytest.mark.parametrize("B,T,nq,nkv,lo,hi", [(1, 64, 32, 8, 4100, 4100), (8, 8, 32, 8, 0, 1600), (64, 2, 16, 8, 1, 700),
                                              (2, 64, 64, 8, 3000, 9001), (1, 1, 32, 8, 20011, 20011),
                                              (3, 16, 40, 8, 5000, 5003)])
def test_attention_serving_sizes(lib, B, T, nq, nkv, lo, hi):
    rnd = random.Random(B)
    c = Attn(lib, [lo, hi][:B] + [rnd.randint(lo, hi) for _ in range(B - 2)], T, nq, nkv, 128, "short", seed=B * T)
    c.run()
    c.check(range(min(B, 6)))


@pytest.mark.parametrize("B,T", [(1, 5), (3, 16), (5, 13), (2, 64)])
def test_attention_fragment_order(lib, B, T):
    c = Attn(lib, [40 + 50 * b for b in range(B)], T, 8, 2, 128, "holes", out_frag=1, seed=B)
    c.run()
    c.check()


def test_attention_values_that_are_not_finite_stay_in_their_branch(lib):
    """Node 2's values are inf / NaN and node 5's key row is NaN: rows that
    see them are not finite, all others are as if those held zeros."""
    par = [-1, 0, 0, 1, 2, 0, 5, 3] + [7] * 32  # 33 nodes and more: two node blocks
    T = len(par)
    c = Attn(lib, [50, 0], T, 8, 2, 128, "chain", splits=2, seed=4)
    c.trees = [par, par]
    c.parents.copy_(i32(c.trees))
    x = c.qkv.view(2, T, 12, 128)
    x[:, 2, 10:, 3] = float("inf")
    x[:, 2, 10:, 4] = NAN
    x[:, 5, 8:10] = NAN
    c.run()
    torch.cuda.synchronize()
    got = c.rows()
    up = tree_oracle.ancestors(par)
    sees2 = torch.tensor([2 in u for u in up], device=DEV)
    sees5 = torch.tensor([5 in u for u in up], device=DEV)
    assert got[:, sees5].isnan().all()
    assert torch.isposinf(got[:, sees2][..., 3]).all() and got[:, sees2][..., 4].isnan().all()
    rest = torch.ones(128, dtype=torch.bool, device=DEV)
    rest[3:5] = False
    assert got[:, sees2][..., rest].isfinite().all()
    clean = ~sees2 & ~sees5
    assert got[:, clean].isfinite().all()
    assert (c.vno.view(2, 2, T, 128)[:, :, 2, 3] == float("inf")).all()
    x[:, 2, 10:, 3:5] = 0
    x[:, 5, 8:10] = 1
    ref = Attn(lib, [50, 0], T, 8, 2, 128, "chain", splits=2, seed=4)
    ref.parents.copy_(i32(c.trees))
    ref.qkv.copy_(c.qkv)
    ref.run()
    torch.cuda.synchronize()
    assert torch.equal(ref.rows()[:, clean], got[:, clean])
    assert torch.equal(ref.rows()[:, sees2][..., rest], got[:, sees2][..., rest])


# Shapes of the many-row kernel: 128 or 256 query rows per workgroup, up to 32 or
# up to 64 nodes, both head sizes; it takes over by what a full cache would cost
# to read, so the capacities are large and the lengths need not be.
WIDE = [(17, 32, 8, 128, 16416, 128), (27, 32, 8, 128, 12256, 128), (64, 16, 8, 128, 12256, 128),
        (20, 64, 8, 128, 10304, 256), (64, 64, 8, 128, 3200, 256), (64, 4, 2, 64, 97728, 128),
        (10, 16, 2, 64, 130400, 128), (33, 16, 2, 64, 45184, 256), (9, 32, 2, 64, 82016, 256)]


def wide(c, group_rows):
    """The call's row groups are the many-row kernel's, as the partials' size shows."""
    rows = c.T * (c.nq // c.nkv)
    a = capi.TreeAttnArgs.from_buffer_copy(c.a)
    a.splits = 2
    groups = -(-rows // group_rows)
    return c.lib.tree_attn_workspace(a)[0] == 4 * c.B * c.nkv * 2 * groups * group_rows * (c.D + 2)


@pytest.mark.parametrize("T,nq,nkv,D,cap,group_rows", WIDE)
def test_attention_many_rows(lib, T, nq, nkv, D, cap, group_rows):
    """Runs of no, one, two, an odd and an even number of blocks, shorter and
    longer than the ring, ragged ends, one workgroup or several."""
    for i, (L, splits) in enumerate([(0, 1), (1, 0), (32, 1), (33, 2), (255, 1), (256, 1), (290, 1), (320, 3), (700, 1),
                                     (737, 1), (1500, 2), (2049, 5), (min(cap - T, 6000), 1), (cap - T, 0)]):
        c = Attn(lib, [L], T, nq, nkv, D, ["holes", "random", "short", "star"][i % 4], splits=splits, seed=i, cap=cap)
        assert wide(c, group_rows)
        c.run()
        c.check()


@pytest.mark.parametrize("T,nq,nkv,cap,group_rows", [(40, 64, 8, 2560, 256), (40, 16, 8, 5600, 128), (17, 32, 8, 5600, 128)])
def test_attention_many_rows_values_that_are_not_finite(lib, T, nq, nkv, cap, group_rows):
    """As above: such a node reaches the rows that see it, and no other."""
    par = ([-1, 0, 0, 1, 2, 0, 5, 3] + [7] * 64)[:T]

    def call():
        c = Attn(lib, [50, 0, 1000], T, nq, nkv, 128, "chain", splits=2, seed=4, cap=cap)
        assert wide(c, group_rows)
        c.trees = [par] * 3
        c.parents.copy_(i32(c.trees))
        return c, c.qkv.view(3, T, nq + 2 * nkv, 128)

    c, x = call()
    x[:, 2, nq + nkv:, 3] = float("inf")
    x[:, 2, nq + nkv:, 4] = NAN
    x[:, 5, nq:nq + nkv] = NAN
    c.run()
    torch.cuda.synchronize()
    up = tree_oracle.ancestors(par)
    sees2 = torch.tensor([2 in u for u in up], device=DEV)
    sees5 = torch.tensor([5 in u for u in up], device=DEV)
    rest = torch.ones(128, dtype=torch.bool, device=DEV)
    rest[3:5] = False
    got = c.rows()
    assert got[:, sees5].isnan().all()
    assert torch.isposinf(got[:, sees2][..., 3]).all() and got[:, sees2][..., 4].isnan().all()
    ref, y = call()
    y.copy_(x)
    y[:, 2, nq + nkv:, 3:5] = 0
    y[:, 5, nq:nq + nkv] = 1
    ref.run()
    torch.cuda.synchronize()
    assert got[:, sees2][..., rest].isfinite().all() and got[:, ~sees2 & ~sees5].isfinite().all()
    assert torch.equal(ref.rows()[:, ~sees2 & ~sees5], got[:, ~sees2 & ~sees5])
    assert torch.equal(ref.rows()[:, sees2][..., rest], got[:, sees2][..., rest])


@pytest.mark.parametrize("T,nq,nkv,cap", [(4, 8, 2, 512), (40, 8, 2, 512), (64, 64, 8, 6304)])
@pytest.mark.parametrize("splits", [1, 2, 3])
def test_attention_scores_that_overflow(lib, T, nq, nkv, cap, splits):
    """Every score between nodes is -inf.  Beside cached keys of score 0 a node has
    weight 0 and a row is the mean of the cached values; with scores of -inf
    everywhere it is NaN, as the softmax is, in one split as in several."""
    c = Attn(lib, [300], T, nq, nkv, 128, "holes", splits=splits, seed=T, cap=cap)
    c.qkv.view(T, nq + 2 * nkv, 128)[c.live, :nq + nkv] = 1
    c.qn.fill_(1e20)
    c.kn.fill_(-1e20)
    c.cos.fill_(1)
    c.sin.fill_(0)
    c.k[:, :, :300] = 0
    c.run()
    torch.cuda.synchronize()
    got = c.rows()[0].double()
    v = c.v_rows[0, :, :300].double()
    ref = v.mean(1).repeat_interleave(nq // nkv, 0)
    mag = v.abs().mean(1).repeat_interleave(nq // nkv, 0)
    assert (got[~c.live] == 0).all()
    assert ((got[c.live] - ref).abs() <= bound(ref, mag, 300, T)).all()
    c.k[:, :, :300] = -1e20
    c.run()
    torch.cuda.synchronize()
    assert c.rows()[0][c.live].isnan().all() and (c.rows()[0][~c.live] == 0).all()


@pytest.mark.parametrize("L", [-1, -(1 << 31), 57, 64, (1 << 31) - 1])
@pytest.mark.parametrize("splits", [1, 4])
def test_attention_invalid_length(lib, L, splits):
    """cap 64 and 8 nodes: a length past 56 is refused on the device."""
    c = Attn(lib, [20, 56, 30], 8, 8, 2, 128, "random", splits=splits, cap=64)
    c.lens.copy_(i32([20, L, 30]))
    c.run()
    torch.cuda.synchronize()
    assert c.rows()[1].isnan().all()
    assert (c.kno[1] == 7).all() and (c.vno[1] == 7).all()
    c.check([0, 2])


def rows_and_terms(c, b, heads):
    """Float64 keys of sequence b's chain and the sum of the absolute values of
    the rotation's two terms."""
    L, T, D = c.lens_l[b], c.T, c.D
    x = c.qkv[b * T:(b + 1) * T].view(T, -1, D)[:, heads].double()
    cos, sin = c.cos[L:L + T, None].double(), c.sin[L:L + T, None].double()
    k = tree_oracle.head_norm_rope(x, c.kn.double(), cos, sin, EPS)
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * c.kn.double()
    half = torch.cat((y[..., D // 2:], y[..., :D // 2]), -1)
    return k.transpose(0, 1), ((y * cos).abs() + (half * sin).abs()).transpose(0, 1)


@pytest.mark.parametrize("D,nq,nkv", [(128, 32, 8), (64, 8, 2)])
@pytest.mark.parametrize("T", [8, 64])
def test_attention_real_rows_and_tables(lib, D, nq, nkv, T):
    """Ordinary rows: keys within half a bf16 step of the formula (and its fp32
    terms), outputs within what one rounding of every query and key entry can
    do to the scores, 2 * 2^-8 * sum |q k| / sqrt(D), twice (numerator and
    denominator); the mean error is 50 times below that bound."""
    lens = [0, 333, 600]
    c = Attn(lib, lens, T, nq, nkv, D, "chain", cap=704, seed=2)
    c.qkv.normal_(generator=torch.Generator(device=DEV).manual_seed(1))
    c.cos, c.sin = rope(704, D)
    c.a.cos_tab, c.a.sin_tab = c.cos.data_ptr(), c.sin.data_ptr()
    c.run()
    torch.cuda.synchronize()
    for b, L in enumerate(lens):
        k, terms = rows_and_terms(c, b, slice(nq, nq + nkv))
        assert ((c.kno[b].double() - k).abs() <= k.abs() * 2.0 ** -8 + terms * 2.0 ** -20).all()
        ref, mag, kn, vn = tree_oracle.attention(c.qkv[b * T:(b + 1) * T], c.trees[b], L, c.k[b], c.v_rows[b], c.qn, c.kn,
                                                 c.cos, c.sin, nq, nkv, EPS)
        assert torch.equal(c.vno[b].double(), vn)
        err = (c.rows()[b].double() - ref).abs()
        qk = max(float(c.kn.double().abs().max()), float(c.k[b, :, :L].double().abs().max()) if L else 0) * D ** 0.5
        limit = bound(ref, mag, L, T) + mag * 4 * 2.0 ** -8 * qk
        assert (err <= limit).all() and err.mean() <= limit.mean() / 50


def test_attention_chain_against_the_decode_attention(lib):
    """A chain's keys and values against what qdec_attn writes to the cache:
    the same values; keys within its extra roundings (two of a normalised entry,
    one of each term, 3 * 2^-8 of the terms, and a half step each of the sum)."""
    B, T, nq, nkv, D, cap = 3, 8, 32, 8, 128, 640
    lens = [0, 333, 600]
    c = Attn(lib, lens, T, nq, nkv, D, "chain", cap=cap, seed=2)
    c.qkv.normal_(generator=torch.Generator(device=DEV).manual_seed(1))
    c.cos, c.sin = rope(cap, D)
    c.a.cos_tab, c.a.sin_tab = c.cos.data_ptr(), c.sin.data_ptr()
    c.run()
    k, v = c.k.clone(), c.v.clone()
    out = torch.zeros((B * T, nq * D), dtype=torch.bfloat16, device=DEV)
    a = capi.AttnArgs(eps=EPS, sm_scale=D ** -0.5, batch=B, t_rows=T, nq=nq, nkv=nkv, head_dim=D, cap=cap, chunk=cap,
                      waves=4)
    for f, t in (("qkv", c.qkv), ("q_norm_w", c.qn), ("k_norm_w", c.kn), ("cos_tab", c.cos), ("sin_tab", c.sin),
                 ("lens", c.lens), ("k_cache", k), ("v_cache", v), ("out", out)):
        setattr(a, f, t.data_ptr())
    lib.attn(a, stream())
    torch.cuda.synchronize()
    vr = v.transpose(-1, -2).reshape(B, nkv, cap, D)
    for b, L in enumerate(lens):
        ref, terms = rows_and_terms(c, b, slice(nq, nq + nkv))
        diff = (c.kno[b].double() - k[b, :, L:L + T].double()).abs()
        assert (diff <= terms * (3 * 2.0 ** -8 + 2.0 ** -15) + ref.abs() * (2 * 2.0 ** -8)).all()
        assert torch.equal(c.vno[b].view(torch.int16), vr[b, :, L:L + T].view(torch.int16))


def test_attention_offsets_past_32_bits(lib):
    """The last sequence's slab starts 3.2 Gi elements into each cache."""
    B, T, nq, nkv, D, cap = 4, 6, 2, 1, 128, 1 << 23
    assert (B - 1) * nkv * cap * D > 1 << 31
    small = Attn(lib, [300], T, nq, nkv, D, "random", splits=3, cap=512, seed=9)
    k = torch.empty((B, nkv, cap, D), dtype=torch.bfloat16, device=DEV)
    v = torch.empty((B, nkv, cap // 8, D, 8), dtype=torch.bfloat16, device=DEV)
    k[B - 1, :, :512], v[B - 1, :, :64] = small.k[0], small.v[0]
    lens = i32([0, 0, 0, 300])
    par = i32([small.trees[0]] * B)
    qkv = small.qkv.repeat(B, 1)
    cos = torch.zeros((cap, D), dtype=torch.bfloat16, device=DEV)
    sin = torch.zeros_like(cos)
    cos[:512], sin[:512] = small.cos, small.sin
    kno, vno = (torch.zeros((B, nkv, T, D), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    out = torch.zeros((B * T, nq * D), dtype=torch.bfloat16, device=DEV)
    a = capi.TreeAttnArgs()
    for f, t in (("qkv", qkv), ("q_norm_w", small.qn), ("k_norm_w", small.kn), ("cos_tab", cos), ("sin_tab", sin),
                 ("lens", lens), ("parents", par), ("k_cache", k), ("v_cache", v), ("k_nodes", kno), ("v_nodes", vno),
                 ("out", out)):
        setattr(a, f, t.data_ptr())
    a.eps, a.sm_scale, a.batch, a.t_rows, a.nq, a.nkv, a.head_dim, a.cap, a.splits = EPS, D ** -0.5, B, T, nq, nkv, D, cap, 3
    pb, cb = lib.tree_attn_workspace(a)
    part = torch.zeros((pb // 4,), device=DEV)
    a.partial = part.data_ptr()
    lib.tree_attn(a, stream())
    small.run()
    small.check()
    assert torch.equal(out.view(B, T, -1)[3], small.out[:T]) and torch.equal(kno[3], small.kno[0])
    # and the accepted path goes to that slab
    c = capi.TreeCommitArgs()
    path, acc, after = i32([[0] + [-1] * (T - 1)] * B), i32([0] * B), i32([1, 1, 1, 301])
    for f, t in (("k_nodes", kno), ("v_nodes", vno), ("k_cache", k), ("v_cache", v), ("path", path), ("naccept", acc),
                 ("lens", after)):
        setattr(c, f, t.data_ptr())
    c.n_layers, c.batch, c.t_rows, c.nkv, c.head_dim, c.cap = 1, B, T, nkv, D, cap
    lib.tree_commit(c, stream())
    torch.cuda.synchronize()
    assert torch.equal(k[3, :, 300], kno[3, :, 0]) and torch.equal(v[3, :, 37, :, 4], vno[3, :, 0])
    del k, v
    torch.cuda.empty_cache()


def test_attention_in_a_graph_and_on_another_stream(lib):
    """One captured call replayed with lengths and trees that change between
    the replays, eager work on the same tensors in between."""
    c = Attn(lib, [70, 0, 200], 12, 8, 2, 128, "random", splits=4, cap=512, seed=6)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.run()
    torch.cuda.current_stream().wait_stream(side)
    c.check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.run()
    for seed in range(4):
        n = Attn(lib, [10 + 90 * seed, 31 * seed, 480], 12, 8, 2, 128, "holes", splits=4, cap=512, seed=20 + seed)
        n.run()
        n.check()
        for name in ("qkv", "qn", "kn", "cos", "sin", "k", "v", "lens", "parents"):
            getattr(c, name).copy_(getattr(n, name))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(c.out, n.out)


# ------------------------------------------------------------------ drafter


def run_draft(lib, hists, lens, T, primary, backoff, depth, matches):
    B, cap = len(hists), len(hists[0])
    hist, ln = i64(hists), i32(lens)
    ids = torch.full((B * T + 8,), 5, dtype=torch.int64, device=DEV)
    par = torch.full((B * T + 8,), 5, dtype=torch.int32, device=DEV)
    a = capi.TreeDraftArgs(hist=hist.data_ptr(), lens=ln.data_ptr(), ids=ids.data_ptr(), parents=par.data_ptr(),
                           batch=B, cap=cap, t_rows=T, primary=primary, backoff=backoff, depth=depth, matches=matches)
    lib.tree_draft(a, stream())
    torch.cuda.synchronize()
    assert (ids[B * T:] == 5).all() and (par[B * T:] == 5).all()
    return ids[:B * T].view(B, T).tolist(), par[:B * T].view(B, T).tolist()


@pytest.mark.parametrize("vocab", [1, 2, 4, 30])
@pytest.mark.parametrize("T,primary,backoff,depth,matches", [(1, 3, 2, 4, 4), (2, 1, 1, 1, 1), (16, 3, 2, 8, 16),
                                                            (64, 2, 1, 63, 32), (33, 1, 4, 5, 7), (9, 12, 3, 6, 32),
                                                            (64, 64, 5, 2, 32)])
def test_draft(lib, vocab, T, primary, backoff, depth, matches):
    rnd = random.Random(vocab * T)
    cap = 300
    hists = [[rnd.randrange(vocab) - (1 << 40) * (b % 2) for _ in range(cap)] for b in range(24)]
    lens = [0, 1, 2, 3, 4, 12, 63, 64, 65, 128, 299, 298] + [rnd.randrange(cap) for _ in range(10)] + [-5, 4000]
    ids, par = run_draft(lib, hists, lens, T, primary, backoff, depth, matches)
    for b in range(24):
        assert (ids[b], par[b]) == tree_oracle.draft(hists[b], lens[b], T, primary, backoff, depth, matches), (b, lens[b])


@pytest.mark.parametrize("L", [4095, 4096, 4097, 8192, 12289, 32000])
def test_draft_long_history(lib, L):
    """Occurrences on both sides of every scan window's border and at the ends."""
    rnd = random.Random(L)
    cap = L + 5
    h = [rnd.randrange(1 << 20) + 10 for _ in range(cap)]
    at = [2, L - 1] + [L - 1 - w * 4096 + d for w in range(1, 9) for d in (-1, 0, 2) if L - 1 - w * 4096 + d > 8]
    for e in at:
        h[e - 2:e + 1] = [1, 2, 3]
    h[L - 2:L + 1] = [1, 2, 3]
    for matches in (1, 5, 32):
        ids, par = run_draft(lib, [h], [L], 64, 3, 2, 4, matches)
        assert (ids[0], par[0]) == tree_oracle.draft(h, L, 64, 3, 2, 4, matches)


# --------------------------------------------------------------- acceptance


@pytest.mark.parametrize("B,T,vocab", [(1, 1, 2), (5, 2, 2), (40, 7, 2), (33, 16, 3), (9, 63, 2), (9, 64, 2)])
@pytest.mark.parametrize("alias,with_emit", [(False, True), (True, False)])
def test_accept(lib, B, T, vocab, alias, with_emit):
    rnd = random.Random(B * T)
    cap = 50
    trees = [tree(rnd.choice(["chain", "star", "random", "holes", "short"]), T, rnd) for _ in range(B)]
    ids_l = [[rnd.randrange(vocab) + (1 << 33) * (b % 2) for _ in range(T)] for b in range(B)]
    pick_l = [[rnd.randrange(vocab) + (1 << 33) * (b % 2) for _ in range(T)] for b in range(B)]
    hist_l = [[rnd.randrange(9) for _ in range(cap)] for _ in range(B)]
    lens_l = [rnd.randint(0, 60) if b else 48 for b in range(B)]  # some past cap: appended tokens are dropped
    ids, pick, hist, lens, par = i64(ids_l), i64(pick_l), i64(hist_l), i32(lens_l), i32(trees)
    lens_out = lens if alias else torch.full_like(lens, -3)
    acc, path = torch.full_like(lens, -3), torch.full((B, T), -3, dtype=torch.int32, device=DEV)
    emit = torch.full((B, T), -3, dtype=torch.int64, device=DEV)
    a = capi.TreeAcceptArgs(out_tok=pick.data_ptr(), ids=ids.data_ptr(), parents=par.data_ptr(), hist=hist.data_ptr(),
                            lens=lens.data_ptr(), lens_out=lens_out.data_ptr(), naccept=acc.data_ptr(),
                            path=path.data_ptr(), emit=emit.data_ptr() if with_emit else None, batch=B, cap=cap,
                            t_rows=T, stop_len=49)
    lib.tree_accept(a, stream())
    torch.cuda.synchronize()
    for b in range(B):
        # a parent that is out of order is no node's and matches no walk
        p, L = tree_oracle.accept(pick_l[b], ids_l[b], trees[b], hist_l[b], lens_l[b], 49)
        pad = [-1] * (T - len(p))
        assert path[b].tolist() == p + pad and int(acc[b]) == max(len(p) - 1, 0) and int(lens_out[b]) == L
        assert hist[b].tolist() == hist_l[b]
        assert emit[b].tolist() == ([pick_l[b][t] for t in p] + pad if with_emit else [-3] * T)


# ------------------------------------------------------------------- commit


@pytest.mark.parametrize("T,nkv,D,layers", [(1, 2, 64, 3), (5, 3, 128, 2), (64, 2, 128, 2), (64, 1, 64, 5), (16, 8, 128, 4)])
def test_commit(lib, T, nkv, D, layers):
    rnd = random.Random(T * nkv)
    g = torch.Generator(device=DEV).manual_seed(T)
    cap = 160
    # length, path, naccept: every alignment of the first slot, whole and empty paths, and what is refused
    seqs = []
    for i in range(10):
        n = rnd.randint(1, T) if i else T
        seqs.append((rnd.randint(n, cap) if i > 1 else (n if i else cap), [0] + sorted(rnd.sample(range(1, T), n - 1)), n - 1))
    seqs += [(40, [-1] * T, 0),  # frozen
             (40, [0, T][:T], min(1, T - 1)) if T > 1 else (40, [-1], 0), (40, [0, -2][:T] if T > 1 else [-1], min(1, T - 1)),
             (cap + 1, [0], 0), (0, [0], 0), (-(1 << 31), [0], 0), ((1 << 31) - 1, [0], 0), (40, list(range(T)), T), (40, [0], (1 << 31) - 1), (40, [0], -1), (40, [1] if T > 1 else [-1], 0)]
    B = len(seqs)
    kn, vn = (torch.randn((layers, B, nkv, T, D), generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
    k = torch.randn((layers, B, nkv, cap, D), generator=g, device=DEV).to(torch.bfloat16)
    vr = torch.randn((layers, B, nkv, cap, D), generator=g, device=DEV).to(torch.bfloat16)
    v = v_layout(vr)
    path = i32([p + [-1] * (T - len(p)) for _, p, _ in seqs])
    acc, lens = i32([a for _, _, a in seqs]), i32([L for L, _, _ in seqs])
    a = capi.TreeCommitArgs(k_nodes=kn.data_ptr(), v_nodes=vn.data_ptr(), k_cache=k.data_ptr(), v_cache=v.data_ptr(),
                            path=path.data_ptr(), naccept=acc.data_ptr(), lens=lens.data_ptr(), n_layers=layers,
                            batch=B, t_rows=T, nkv=nkv, head_dim=D, cap=cap)
    want_k, want_v = k.clone(), vr.clone()
    for b, (L, p, n) in enumerate(seqs[:10]):
        for i, t in enumerate(p):
            want_k[:, b, :, L - len(p) + i], want_v[:, b, :, L - len(p) + i] = kn[:, b, :, t], vn[:, b, :, t]
    lib.tree_commit(a, stream())
    torch.cuda.synchronize()
    assert torch.equal(k, want_k) and torch.equal(v, v_layout(want_v))
