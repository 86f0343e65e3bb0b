"""The 8-bit cache over the whole range of its numbers: what is finite stays finite, at the
largest and the smallest scales, scores, queries and values that fp32 holds.

Where scores are large, their rounding is too, so the cases are those whose result does not
depend on it: scores that are the same number for every slot (weights exactly equal),
or so far apart that one slot has all the weight (the next one less than e^-100).  What is left
of the tolerance of test_kv8_gpu.py is then its part without scores:
  2^-8 |ref|  the rounding to bf16, and of mag = sum |p v| / sum p
  2^-11       w = p * v_scale in fp16
  (n + 64) 2^-22  sums over n slots, exponentials, rescaling factors in fp32
and 2^-39 step for fp16's smallest steps."""

import math

import pytest
import torch

from oracle import kv8_oracle as ko
from qdec import capi
from test_kv8_gpu import BF, DEV, EPS, NAN, Call, cache, gen, lib, ptrs, randn, slab, stream  # noqa: F401  (lib: the fixture)

pytestmark = pytest.mark.gpu


def read_back(lib, c, B, nkv, D, cap, n):
    """Slots 0 .. n - 1 of a cache as rows of bf16."""
    slots = (n + 31) // 32 * 32
    k, v = torch.zeros((B, nkv, slots, D), dtype=BF, device=DEV), torch.zeros((B, nkv, slots // 8, D, 8), dtype=BF, device=DEV)
    lib.kv8_load(capi.Kv8LoadArgs(k_slab=k.data_ptr(), v_slab=v.data_ptr(), batch=B, nkv=nkv, head_dim=D, cap=cap, slab_cap=slots,
                                  n=n, **ptrs(c)), stream())
    return k[:, :, :n], ko.slab_rows(v)[:, :, :n]


@pytest.mark.parametrize("D", [128, 64])
def test_load_of_any_scale(lib, D):
    B, nkv, cap = 2, 3, 192
    c = cache(gen(3), B, nkv, cap, D)
    c["k8"].clamp_(min=-127), c["v8"].clamp_(min=-127)  # what a store writes
    big = torch.tensor([0x7f7f, 0x7f7e, 0x7f7d, 0x7f00], dtype=torch.int16).view(BF).double()
    scales = torch.cat(((big / 127).float(), torch.tensor([2.0 ** 120, 2.0 ** -100 / 127, 2.0 ** -100, 0.0, NAN, 1e-20, 1.0])))
    for name in ("k_scale", "v_scale"):
        c[name].copy_(scales.to(DEV)[torch.randint(len(scales), (B, nkv, cap), generator=gen(4), device=DEV)])
    for got, q8, sc in zip(read_back(lib, c, B, nkv, D, cap, cap), (c["k8"], ko.row_major(c["v8"])), (c["k_scale"], c["v_scale"])):
        want = (q8.float() * sc[..., None]).to(BF)
        torch.testing.assert_close(got, want, rtol=0, atol=0, equal_nan=True)
        assert torch.equal(torch.isfinite(got), torch.isfinite(sc)[..., None].expand_as(got))


@pytest.mark.parametrize("D", [128, 64])
def test_extreme_rows_there_and_back(lib, D):
    """Rows whose largest is a bf16 number at either end of what is held."""
    tops = torch.tensor([0x7f7f, 0x7f7e, 0x7f7d, 0x7f01, 0x7f00, 0x7e80, 0x3f80, 0x0e01, 0x0d80, 0x0d7f, 0x0001, 0x0000],
                        dtype=torch.int16, device=DEV).view(BF)  # 0x0d80: 2^-100
    g, n = gen(6), len(tops)
    rows = []
    for _ in range(2):
        x = (torch.rand((1, 2, n, D), generator=g, device=DEV) * 2 - 1) * tops.float()[:, None]
        x[..., 7], x[..., 20] = tops.float(), 0.0
        rows.append(x.to(BF))
    ks, vs = slab(rows, 32)
    c = cache(g, 1, 2, 64, D)
    lib.kv8_store(capi.Kv8StoreArgs(k_slab=ks.data_ptr(), v_slab=vs.data_ptr(), batch=1, nkv=2, head_dim=D, cap=64, slab_cap=32, pos0=0,
                                    n=n, **ptrs(c)), stream())
    for got, x in zip(read_back(lib, c, 1, 2, D, 64, n), rows):
        q, s = ko.hold(x)
        want = (q.float() * s.float()[..., None]).to(BF)
        assert bool(torch.isfinite(got).all()) and bool((got[..., 20] == 0).all())
        assert torch.equal(got, want)


def along_one_channel(lib, shape, splits, gain, key):
    """A call whose queries lie on channel 63 alone, so that a slot's score is gain times
    its key there: 100 * key(slot), and 0 for the new slots."""
    B, nq, nkv, D, T, lens = shape
    a = Call(lib, *shape, splits=splits)
    x = a.qkv.view(B * T, -1, D)
    x[:, :nq] = 0.0
    x[:, :nq, D // 2 - 1] = 1.0
    x[:, nq:nq + nkv, D // 2 - 1] = 0.0
    a.cos[:], a.sin[:] = 1.0, 0.0
    a.qw[D // 2 - 1] = gain
    a.c["k8"][..., D // 2 - 1] = 100
    for b, L in enumerate(lens):
        a.c["k_scale"][b, :, :L] = key(torch.arange(L, device=DEV, dtype=torch.float32), L)
    return a


def check_no_score_error(a, score=0.0, least=0.0):
    """`score`: what is known of the weights' error all the same, `least`: an error of any output."""
    a.run()
    got, tab = a.rows().double(), (a.cos[:a.T], a.sin[:a.T])
    assert bool(torch.isfinite(got).all())
    for b, L in enumerate(a.lens):
        q = ko.norm_rope(a.qkv.view(a.B, a.T, a.nq + 2 * a.nkv, a.D)[b, :, :a.nq], a.qw, *tab, EPS)
        ref, mag, step, _, _ = ko.attend(q, a.c["k8"][b], a.c["k_scale"][b], a.c["v8"][b], a.c["v_scale"][b], L, a.D ** -0.5)
        tol = 2 ** -8 * ref.abs() + mag * (2 ** -11 + score + (L + a.T + 64) * 2 ** -22) + step * 2 ** -39 + least
        worst = ((got[b] - ref).abs() / tol).max().item()
        assert worst <= 1, f"sequence {b} of length {L}: {worst:.3g} of the tolerance"


SHAPES = [(1, 32, 8, 128, 1, [900]), (2, 32, 8, 128, 2, [700, 61]), (1, 32, 8, 128, 9, [1500]), (2, 8, 2, 64, 3, [64, 1100]),
          (9, 16, 8, 128, 4, [55 * i + 1 for i in range(9)]), (3, 64, 8, 128, 8, [2000, 511, 5])]
ORDERS = {
    "equal": lambda i, L: torch.full_like(i, 0.01),
    "rising": lambda i, L: 0.001 * (i + 1),
    "falling": lambda i, L: 0.001 * (L - i),
    "mixed": lambda i, L: 0.001 * (1 + (i * 641) % L if math.gcd(641, L) == 1 else 1 + i),
}


@pytest.mark.parametrize("shape", SHAPES, ids=[f"{s[0]}x{s[1]}/{s[2]}x{s[3]}-t{s[4]}" for s in SHAPES])
@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("order", sorted(ORDERS))
def test_scores_of_any_size(lib, shape, splits, order):
    """gain times 1 for every slot, or gain / 10 from one to the next."""
    for log2 in (10, 20, 24, 25, 26, 27, 30, 31, 33, 40, 60, 100):
        check_no_score_error(along_one_channel(lib, shape, splits, 2.0 ** log2, ORDERS[order]))


@pytest.mark.parametrize("shape", SHAPES, ids=[f"{s[0]}x{s[1]}/{s[2]}x{s[3]}-t{s[4]}" for s in SHAPES])
@pytest.mark.parametrize("log2", [20, 24, 28, 32, 50, 90])
def test_large_random_scores_stay_among_the_values(lib, shape, log2):
    """An output is a mean of values: never beyond the largest of them, by more than the
    rounding of the weights (2^-11) and its own (2^-8)."""
    a = Call(lib, *shape, gain=2.0 ** log2).run()
    got = a.rows()
    assert bool(torch.isfinite(got).all())
    for b, L in enumerate(a.lens):
        end = L + a.T
        top = (ko.row_major(a.c["v8"])[b, :, :end].float().abs() * a.c["v_scale"][b, :, :end, None]).amax((1, 2))  # per kv head
        most = got[b].float().abs().view(a.T, a.nkv, -1).amax((0, 2))
        assert bool((most <= top * (1 + 2 ** -7)).all())


@pytest.mark.parametrize("shape", SHAPES, ids=[f"{s[0]}x{s[1]}/{s[2]}x{s[3]}-t{s[4]}" for s in SHAPES])
@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("log2", [-60, -80, -86, -92, 110, 120])
def test_values_of_one_size(lib, shape, splits, log2):
    """All values, the new ones too, about 2^log2: from near 2^-100, where rows are held as
    zeros, to near the largest bf16 number."""
    a = Call(lib, *shape, splits=splits)
    a.c["v_scale"].copy_((torch.rand(a.c["v_scale"].shape, generator=gen(8), device=DEV) * 0.01 + 0.002) * 2.0 ** log2)
    a.qkv.view(a.B * a.T, -1, a.D)[:, -a.nkv:] *= 2.0 ** log2
    a.checked()
    assert bool((a.rows().float().abs().amax(-1) > 2.0 ** (log2 - 12)).all())


@pytest.mark.parametrize("shape", SHAPES, ids=[f"{s[0]}x{s[1]}/{s[2]}x{s[3]}-t{s[4]}" for s in SHAPES])
@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("gap", [60.0, 75.0, 80.0, 84.0])
def test_small_weights_beside_values_of_zero(lib, shape, splits, gap):
    """The last cached slot has values of zero and a score `gap` above all others, so an output
    is their values times e^-gap, down to 2^-121.  The one score is off by its query's 21
    bits (2^-20 of it) and by 64 roundings at most, which scales every other weight; an output
    is held times 2^-20 (in up to 3 partials), so in steps of 2^-129, rounded once each and
    once where it is joined."""
    a = along_one_channel(lib, shape, splits, 1.0, lambda i, L: torch.where(i == L - 1, gap / 100, 0.0))
    a.c["v_scale"].copy_(torch.rand(a.c["v_scale"].shape, generator=gen(8), device=DEV) * 5 + 1)
    for b, L in enumerate(a.lens):
        a.c["v_scale"][b, :, L - 1] = 0.0
    check_no_score_error(a, score=2 * gap * (2 ** -20 + 64 * 2 ** -24), least=6 * 2.0 ** -130)
    assert bool((a.rows().float().abs().amax(-1) > 2.0 ** -126).all())


@pytest.mark.parametrize("shape", SHAPES, ids=[f"{s[0]}x{s[1]}/{s[2]}x{s[3]}-t{s[4]}" for s in SHAPES])
@pytest.mark.parametrize("order", sorted(ORDERS))
def test_queries_up_to_the_largest_number(lib, shape, order):
    """Queries whose one channel is gain sqrt(D), from just below 2^127 to just below 2^128 (eps
    takes it below), beside keys of 2^-100."""
    for gain in {128: [1.0, 1.375], 64: [1.0, 2.0]}[shape[3]]:
        check_no_score_error(along_one_channel(lib, shape, 1, gain * 2.0 ** 124, lambda i, L: ORDERS[order](i, L) * 2.0 ** -100))


@pytest.mark.parametrize("shape", SHAPES, ids=[f"{s[0]}x{s[1]}/{s[2]}x{s[3]}-t{s[4]}" for s in SHAPES])
@pytest.mark.parametrize("sm_scale", [1e-10, 1e-20, 1e-38])
def test_zero_queries_under_a_tiny_scale(lib, shape, sm_scale):
    """Scores of 0 for every slot: the values' mean."""
    a = along_one_channel(lib, shape, 1, 1.0, ORDERS["mixed"])
    a.qkv.view(a.B * a.T, -1, a.D)[:, :a.nq] = 0.0
    a.a.sm_scale = sm_scale
    check_no_score_error(a)


@pytest.mark.parametrize("shape", [(5, 40, 8, 128, 1, [639, 0, 1500, 64, 512]), (3, 9, 3, 64, 5, [59, 1123, 0]),
                                   (2, 1, 1, 64, 1, [700, 300]), (2, 7, 7, 128, 1, [900, 3])])
@pytest.mark.parametrize("splits", [2, 3])
def test_partials_of_an_odd_number_of_rows(lib, shape, splits):
    """Every split's partial begins at a multiple of 16 bytes; what out_partials leaves, merged
    in 64 bits, against the call's own rows: both round once to bf16."""
    B, nq, nkv, D, T, lens = shape
    R = T * nq // nkv
    assert R % 2
    a, b = Call(lib, *shape, splits=splits).run(), Call(lib, *shape, splits=splits)
    b.a.out_partials = 1
    b.partial.fill_(NAN)
    b.run()
    pb, stride = lib.kv8_attn_workspace(b.a)[0], R * (D + 2) + 2
    assert pb == 4 * B * nkv * splits * stride and stride % 4 == 0
    part = b.partial[:pb // 4].view(B, nkv, splits, stride).double()
    acc, m, l, pad = part[..., :R * D].reshape(B, nkv, splits, R, D), part[..., R * D:R * (D + 1)], part[..., R * (D + 1):-2], part[..., -2:]
    assert bool(torch.isnan(pad).all()) and bool(torch.isnan(b.partial[pb // 4:]).all())
    left = ~torch.isnan(m)
    top = m.masked_fill(~left, -math.inf).amax(2, keepdim=True)
    w = torch.where(left, torch.exp2(m - top), 0.0)
    want = (torch.where(w[..., None] > 0, acc, 0.0) * w[..., None]).sum(2) / (torch.where(w > 0, l, 0.0) * w).sum(2)[..., None]
    want = want.view(B, nkv, T, nq // nkv, D).transpose(1, 2).reshape(B, T, nq, D)
    torch.testing.assert_close(a.rows().double(), want, rtol=2 ** -8, atol=float(want.abs().max()) * 2 ** -18)
