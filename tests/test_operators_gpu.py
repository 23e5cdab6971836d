"""The operators of a decoding step against plain 64-bit implementations (tests/operators_ref.py).

Tolerances.  eps = 2^-24 is half a step of 32 bits, h the output type's.  A sum of n products in 32 bits strays from the exact sum by
about sqrt(n) eps times the sum of the products' magnitudes where the roundings are to nearest; a tensor core cuts its sums off
instead, so n / 16 additions (of 16 products) may add up to n / 16 * 2 eps.  The tests allow (8 + sqrt(n) + n / 16) 2 eps.
Attention: a score that is off by t changes a weight by a factor 1 + t, so the output by at most 2 t max|v|; the weights' sum and the
weighted sum add as much as a sum of S products; with 16-bit operands the weights are rounded to half precision (2^-11).
Whole numbers, codes and scales are equal.
"""
import ctypes

import numpy as np
import pytest
import torch

from tests import operators_ref as ref

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24


@pytest.fixture(scope="module")
def api():
    from zoph_rnn_b200 import api as a
    return a


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype="f32"):
    return torch.randn(shape, generator=g, device="cuda").to(ref.TYPES[dtype])


def f64(t):
    return t.detach().double().cpu().numpy()


def sum_tol(n):
    return (8 + n ** 0.5 + n / 16) * 2 * EPS


# ------------------------------------------------------------------ memory4: pack, unpack
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("S, B, heads, d", [(1, 1, 1, 1), (1, 3, 1, 31), (5, 2, 1, 32), (7, 3, 1, 33), (3, 5, 4, 20), (50, 4, 1, 1000), (9, 2, 16, 64), (2, 3, 2, 251), (4, 1, 1, 2048)])
def test_pack_and_unpack(api, dtype, S, B, heads, d):
    g = gen(S + 7 * d)
    x = randn(g, S, B, heads * d, dtype=dtype)
    x[0, 0, : d // 2] *= 1e-3
    m = api.memory4(B, S, d, heads=heads).pack(x)
    codes, scales = ref.pack(f64(x), heads, d)
    np.testing.assert_array_equal(m.scales.cpu().numpy().view(np.uint16), scales.view(np.uint16))
    np.testing.assert_array_equal(m.codes.cpu().numpy(), codes)
    for t in ("f32", "bf16", "f16"):
        want = torch.from_numpy(ref.unpack(codes, scales, d)).to(ref.TYPES[t])
        assert torch.equal(m.unpack(ref.TYPES[t]).cpu(), want)


def test_codes_next_to_the_middle_between_two(api):
    """Quotients that 32 bits round onto k + 1/2 from either side, and exact ties."""
    s = np.float16(0.0123)
    rows = []
    for k in range(-7, 7):
        mid = (k + 0.5) * float(s)  # exact in 32 bits
        f = np.float32(mid)
        rows += [f, np.nextafter(f, np.float32(-9)), np.nextafter(f, np.float32(9))]
    x = np.zeros((1, len(rows), 32), np.float32)
    x[0, :, 0] = rows
    x[0, :, 1] = np.float32(7 * float(s))  # the group's largest: its scale is s
    m = api.memory4(len(rows), 1, 32).pack(torch.from_numpy(x).cuda())
    codes, scales = ref.pack(x.astype(np.float64), 1, 32)
    assert (scales == s).all()
    np.testing.assert_array_equal(m.codes.cpu().numpy(), codes)


@pytest.mark.parametrize("first", [0x2000, 0x0001, 0x6c00])
def test_codes_next_to_the_middle_for_every_mantissa_of_a_scale(api, first):
    """Scales of 2^-7 .. 2^-6, of the subnormal ones, of 4096 .. 8192: numbers on the middle between two codes and next to it."""
    s = np.arange(first, first + 1024 - (first & 1), dtype=np.uint16).view(np.float16).astype(np.float32)
    mid = s[:, None] * (np.arange(-7, 7, dtype=np.float32) + np.float32(0.5))  # (exact: 11 + 4 bits)
    x = np.zeros((1, len(s), 64), np.float32)
    for i, v in enumerate((mid, np.nextafter(mid, np.float32(-1e9)), np.nextafter(mid, np.float32(1e9)))):
        x[0, :, i * 8 : i * 8 + 7] = v[:, :7]
        x[0, :, 32 + i * 8 : 32 + i * 8 + 7] = v[:, 7:]
    x[0, :, 31] = x[0, :, 63] = 7 * s  # the groups' largest
    m = api.memory4(len(s), 1, 64).pack(torch.from_numpy(x).cuda())
    codes, scales = ref.pack(x.astype(np.float64), 1, 64)
    assert (scales.astype(np.float32).reshape(-1, 2) == s[:, None]).all()
    np.testing.assert_array_equal(m.codes.cpu().numpy(), codes)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_ties_of_16_bit_states(api, dtype):
    """Groups whose largest magnitude is a multiple of 7: a good part of the numbers lies on the middle between two codes."""
    g = gen(5)
    x = torch.randint(-28, 29, (40, 6, 320), generator=g, device="cuda").float() * 0.125
    x[..., ::32] = 3.5  # (28 / 8: the scale is 1/2, odd multiples of 1/4 are ties)
    x = (x * 2.0 ** torch.randint(-6, 7, (40, 6, 1), generator=g, device="cuda").float()).to(ref.TYPES[dtype])
    m = api.memory4(6, 40, 320).pack(x)
    codes, scales = ref.pack(f64(x), 1, 320)
    np.testing.assert_array_equal(m.scales.cpu().numpy().view(np.uint16), scales.view(np.uint16))
    np.testing.assert_array_equal(m.codes.cpu().numpy(), codes)


def test_pack_of_numbers_at_the_ends_of_the_range(api):
    x = torch.zeros(1, 10, 64, device="cuda")
    x[0, 0, :32] = 1e-9          # below half precision: zeros
    x[0, 1, :32] = 3e-7          # a scale of a few steps
    x[0, 2, :3] = torch.tensor([1e-7, -4e-7, 2e-7])
    x[0, 3, 5] = 65504.0
    x[0, 4, 5] = -3.0e38         # saturates
    x[0, 5, 40] = float("inf")   # the second group only
    x[0, 6, 3] = float("nan")
    x[0, 7, :] = -0.0
    x[0, 8, 0], x[0, 8, 1] = 1.0, 1e-40
    m = api.memory4(10, 1, 64).pack(x)
    codes, scales = ref.pack(f64(x), 1, 64)
    np.testing.assert_array_equal(m.scales.cpu().numpy().view(np.uint16), scales.view(np.uint16))
    np.testing.assert_array_equal(m.codes.cpu().numpy(), codes)
    v = m.unpack().cpu().reshape(10, 64)
    # (7 * 9352 = 65464, and half precision has steps of 32 there: 65472)
    assert v[4, 5] == -65472 and v[5, :32].eq(0).all() and v[5, 32:].isnan().all() and v[6, :32].isnan().all() and v[9].eq(0).all()


def test_pack_slot_by_slot_leaves_the_others(api):
    g = gen(3)
    x = randn(g, 6, 3, 100)
    whole = api.memory4(3, 6, 100).pack(x)
    m = api.memory4(3, 9, 100)
    m.codes.fill_(77)
    m.scales.fill_(5.0)
    for s in (4, 0, 5, 1, 3, 2):
        m.pack(x[s:s + 1], slot0=s + 2)
    assert torch.equal(m.codes[:, 2:8], whole.codes) and torch.equal(m.scales[:, 2:8], whole.scales)
    assert m.codes[:, :2].eq(77).all() and m.codes[:, 8:].eq(77).all() and m.scales[:, 8:].eq(5).all()
    assert torch.equal(m.unpack(slot0=3, S=2), whole.unpack()[:, 1:3])
    assert m.unpack(slot0=3, S=0).numel() == 0
    wide = torch.randn(6, 3, 128, device="cuda")  # columns and slots further apart than they are long
    wide[..., 9:109] = x
    assert torch.equal(api.memory4(3, 6, 100).pack(wide[..., 9:109]).codes, whole.codes)
    by_col = x.permute(1, 0, 2).contiguous().permute(1, 0, 2)
    assert torch.equal(api.memory4(3, 6, 100).pack(by_col).codes, whole.codes)


# ------------------------------------------------------------------ memory4: attend
def attend_case(api, dtype, B, cols, S, heads, d, lens, offsets, scale=None, seed=0, mask=None, qmul=1.0):
    g = gen(seed)
    hs = torch.tanh(0.5 * torch.randn(S, B, heads * d, generator=g, device="cuda"))
    q = (qmul * torch.tanh(torch.randn(B * cols, heads * d, generator=g, device="cuda"))).to(ref.TYPES[dtype])
    m = api.memory4(B, S, d, heads=heads).pack(hs)
    scale = (1.0 if heads == 1 else d ** -0.5) if scale is None else scale
    ln, of = torch.tensor(lens, dtype=torch.int32, device="cuda"), torch.tensor(offsets, dtype=torch.int32, device="cuda")
    mk = None if mask is None else torch.tensor(mask, dtype=torch.int32, device="cuda")
    out = m.attend(q, ln, of, scale=scale, mask01=mk)
    v = ref.unpack(m.codes.cpu().numpy(), m.scales.cpu().numpy(), d)
    check_attend(out, v, f64(q), lens, offsets, scale, dtype, mask)
    return m, q, ln, of, scale, out


def check_attend(out, v, q, lens, offsets, scale, dtype, mask=None):
    want, mag = ref.attend(v, q, lens, offsets, scale, mask)
    B, S, heads, d = v.shape
    vmax = np.nanmax(np.abs(v))
    n = max([1] + [min(o + l, S) - max(o, 0) for o, l in zip(offsets, lens)])
    tol = vmax * (2 * sum_tol(d) * mag + 4 * sum_tol(n) + (0.0 if dtype == "f32" else 2 * 2.0 ** -11))[..., None] + ref.HALF_STEP[dtype] * np.abs(want)
    # Columns without slots are zeros to the bit.  (Zero queries are none: equal weights p = 1, so out = (sum v) * (1 / n) has two roundings of its own
    # beside the sum's, 2 * 2^-24 |out|, more than the half step that "scores of magnitude 0" would leave.)
    cols = want.shape[0] // B
    empty = [min(int(offsets[c // cols]) + int(lens[c // cols]), S) <= max(int(offsets[c // cols]), 0) or (mask is not None and mask[c] == 0) for c in range(want.shape[0])]
    tol[empty] = 0.0
    err = np.abs(f64(out).reshape(want.shape) - want)
    assert np.isfinite(err).all() and (err <= tol).all(), (err.max(), (err / np.maximum(tol, 1e-300)).max())


@pytest.mark.parametrize("lens", [[0, 0, 0, 0, 0], [0, 4000, 0, 0, 1], [4000, 33, 3999, 65, 1000], [2000] * 5])
def test_attend_over_few_columns_of_very_different_lengths(api, lens):
    """Source columns that share the multiprocessors: none, one or several CTAs' worth of slots each."""
    attend_case(api, "bf16", 5, 3, 4000, 1, 264, lens, [4000 - n for n in lens], seed=sum(lens))
    attend_case(api, "f32", 5, 2, 4000, 1, 72, lens, [0] * 5, seed=sum(lens))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d, S", [(64, 700), (128, 90), (512, 700)])
def test_attend_to_scores_that_rise_or_fall_along_the_window(api, dtype, d, S):
    """Running maxima that rise in many small steps, in a few large ones, or never after the first slots."""
    g = gen(d)
    for span in (12.0, 120.0, -40.0):
        ramp = torch.linspace(0.05, 1.0, S, device="cuda") if span > 0 else torch.linspace(1.0, 0.05, S, device="cuda")
        u = torch.where(torch.rand(d, generator=g, device="cuda") < 0.5, -1.0, 1.0)
        hs = (ramp[:, None, None] * u).expand(S, 2, d).contiguous()
        q = (u * torch.tensor([1.0, 0.5], device="cuda").repeat(2)[:, None]).to(ref.TYPES[dtype])
        m = api.memory4(2, S, d).pack(hs)
        lens = [S, S - 40]
        out = m.attend(q, torch.tensor(lens, dtype=torch.int32, device="cuda"), scale=abs(span) / d)
        check_attend(out, ref.unpack(m.codes.cpu().numpy(), m.scales.cpu().numpy(), d), f64(q), lens, [0, 0], abs(span) / d, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B, cols, S, heads, d", [
    (1, 1, 1, 1, 1), (1, 12, 23, 1, 1000), (3, 5, 33, 1, 100), (2, 12, 64, 1, 512), (4, 1, 31, 1, 320), (2, 17, 65, 1, 1024), (2, 33, 40, 1, 96), (3, 2, 100, 8, 64),
    (2, 4, 129, 4, 33), (1, 3, 700, 2, 128), (1, 16, 3000, 1, 200), (2, 3, 257, 16, 20), (1, 40, 50, 3, 251), (5, 8, 90, 1, 129), (2, 1, 4500, 1, 640)])
def test_attend(api, dtype, B, cols, S, heads, d):
    lens = [max(1, S - 3 * b) for b in range(B)]
    attend_case(api, dtype, B, cols, S, heads, d, lens, [S - n for n in lens], seed=d + S)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B, cols, S, heads, d", [(130, 3, 40, 8, 64), (99, 1, 33, 16, 32), (60, 17, 5, 12, 100), (300, 12, 1, 4, 33), (41, 9, 70, 30, 128), (700, 2, 32, 1, 20)])
def test_attend_with_many_short_heads(api, dtype, B, cols, S, heads, d):
    """More column tiles and heads than multiprocessors: a warp each."""
    rng = np.random.default_rng(d)
    lens = rng.integers(0, S + 1, B).tolist()
    offs = [int(rng.integers(0, S - n + 1)) for n in lens]
    mask = (rng.random(B * cols) < 0.9).astype(np.int32).tolist()
    attend_case(api, dtype, B, cols, S, heads, d, lens, offs, seed=d, mask=mask)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("heads, d", [(1, 1000), (4, 64)])
def test_attend_lengths_and_masks(api, dtype, heads, d):
    """Empty sentences, one slot, windows at either end and in the middle of a tile, windows that stick out, masked columns."""
    S, B, cols = 150, 10, 3
    lens = [0, 1, 150, 1, 32, 33, 31, 400, 20, -5]
    offs = [0, 149, 0, 0, 32, 31, 100, -7, 145, 10]
    mask = [1] * (B * cols)
    mask[7] = mask[8] = mask[20] = 0
    *_, out = attend_case(api, dtype, B, cols, S, heads, d, lens, offs, mask=mask)
    out = out.view(B, cols, -1)
    assert out[0].eq(0).all() and out[9].eq(0).all() and out.view(B * cols, -1)[[7, 8, 20]].eq(0).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads, d, S", [(1, 500, 90), (8, 64, 300)])
def test_what_lies_outside_the_window_is_not_looked_at(api, dtype, heads, d, S):
    B, cols = 3, 4
    lens, offs = [S - 40, 7, 33], [13, S - 7, 40]
    m, q, ln, of, scale, out = attend_case(api, dtype, B, cols, S, heads, d, lens, offs)
    for b in range(B):
        for at in (slice(0, offs[b]), slice(offs[b] + lens[b], S)):
            m.codes[b, at] = 255
            m.scales[b, at] = float("nan")
    assert torch.equal(m.attend(q, ln, of, scale=scale), out)
    # a NaN inside reaches the columns of its sentence and no other
    m.scales[1, offs[1] + 2, 0, 0] = float("nan")
    bad = m.attend(q, ln, of, scale=scale).view(B, cols, heads, d)
    assert bad[1, :, 0].isnan().all() and torch.equal(bad[[0, 2]], out.view(B, cols, heads, d)[[0, 2]])
    assert torch.equal(bad[1, :, 1:], out.view(B, cols, heads, d)[1, :, 1:])


def attend_ways(api, B, cols, S, heads, d):
    """How many bytes of scratch memory an attention asks for: some where several CTAs share a source column, else none."""
    n = ctypes.c_size_t()
    assert api.lib().zrnn_memory4_attend_workspace(B, cols, S, heads, d, ctypes.byref(n)) == 0
    return n.value


# several CTAs per source column (heads of one warp, of two teams, of four), a CTA per source column, a warp per column tile and head
DEALT = [(2, 3, 4000, 2, 64), (3, 4, 4000, 1, 264), (2, 17, 3000, 1, 1000)]
OTHERS = [(3, 4, 90, 1, 500), (2, 5, 100, 1, 128), (40, 5, 70, 8, 64)]


def test_attend_is_shared_by_several_ctas_where_these_tests_mean_it(api):
    for shape in DEALT:
        assert attend_ways(api, *shape) > 0
    for shape in OTHERS:
        assert attend_ways(api, *shape) == 0


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B, cols, S, heads, d", DEALT)
def test_attend_lengths_and_masks_on_several_ctas(api, dtype, B, cols, S, heads, d):
    """Windows that stick out at either end, empty ones, one slot, masked columns."""
    for lens, offs in (([S + 50, 0], [-20, 7]), ([-5, S], [3, 0]), ([1, 33], [S - 1, 31]), ([2 * S, S - 100], [100, 2 * S])):
        lens, offs = (lens + [S // 2])[:B], (offs + [S // 3])[:B]
        mask = [1] * (B * cols)
        mask[1] = mask[-1] = 0
        *_, out = attend_case(api, dtype, B, cols, S, heads, d, lens, offs, mask=mask, seed=d)
        assert out[1].eq(0).all() and out[-1].eq(0).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B, cols, S, heads, d", DEALT + OTHERS)
def test_attend_numbers_that_are_not_finite(api, dtype, B, cols, S, heads, d):
    """softmax of scores among which one is a NaN is NaN: a query that is not finite, a memory all of NaN, and NaNs in a few slots anywhere of a
    window reach the columns that attend to them, and no others; masked columns and columns without slots are zeros."""
    lens, offs = [S] * B, [0] * B
    mask = [1] * (B * cols)
    m, q, ln, of, scale, out = attend_case(api, dtype, B, cols, S, heads, d, lens, offs, seed=d)
    base = out.view(B, cols, heads, d)
    for bad in (float("nan"), float("inf"), float("-inf")):
        q2 = q.clone()
        q2[1, d - 1] = bad  # column 1, head 0
        got = m.attend(q2, ln, of, scale=scale).view(B, cols, heads, d)
        assert got[0, 1, 0].isnan().all()
        got = got.clone()
        got[0, 1, 0] = base[0, 1, 0]
        assert torch.equal(got, base)
        mk = torch.ones(B * cols, dtype=torch.int32, device="cuda")
        mk[1] = 0
        assert m.attend(q2, ln, of, scale=scale, mask01=mk)[1].eq(0).all()
        ln0 = ln.clone()
        ln0[0] = 0
        assert m.attend(q2, ln0, of, scale=scale)[:cols].eq(0).all()
    # NaNs in the memory: all of a sentence, a whole tile of slots, one slot, wherever they lie
    for at in (slice(0, S), slice(0, min(32, S)), slice(max(0, S - 40), S), slice(S // 2, S // 2 + 1), slice(S - 1, S)):
        bad = api.memory4(B, S, d, heads=heads, codes=m.codes, scales=m.scales.clone())
        bad.scales[1, at, 0, -1] = float("nan")
        got = bad.attend(q, ln, of, scale=scale).view(B, cols, heads, d)
        assert got[1, :, 0].isnan().all()
        got = got.clone()
        got[1, :, 0] = base[1, :, 0]
        assert torch.equal(got, base)
    # a NaN among slots whose weights are nothing beside the largest one's
    g = gen(d)
    u = torch.where(torch.rand(heads * d, generator=g, device="cuda") < 0.5, -1.0, 1.0)
    hs = (-u).repeat(S, B, 1)
    hs[S // 5] = u
    far = api.memory4(B, S, d, heads=heads).pack(hs)
    qu = u.to(q.dtype).repeat(B * cols, 1)
    fine = far.attend(qu, ln, of, scale=400.0 / d)
    assert fine.isfinite().all()
    far.scales[0, S - 2, 0, 0] = float("nan")
    got = far.attend(qu, ln, of, scale=400.0 / d).view(B, cols, heads, d)
    assert got[0, :, 0].isnan().all() and torch.equal(got[1:], fine.view(B, cols, heads, d)[1:])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B, cols, S, heads, d", DEALT + OTHERS)
def test_attend_to_scores_that_are_all_minus_infinity(api, dtype, B, cols, S, heads, d):
    """The softmax of such a column is NaN; zeros are for columns without slots."""
    g = gen(d)
    m = api.memory4(B, S, d, heads=heads).pack(torch.full((S, B, heads * d), 0.5, device="cuda"))
    q = torch.tanh(torch.randn(B * cols, heads * d, generator=g, device="cuda")).to(ref.TYPES[dtype])
    ln = torch.full((B,), S, dtype=torch.int32, device="cuda")
    base = m.attend(q, ln)
    q2 = q.clone()
    q2[0, 0] = float("-inf")
    got = m.attend(q2, ln)
    assert got[0, :d].isnan().all() and torch.equal(got[1:], base[1:]) and torch.equal(got[0, d:], base[0, d:])
    mask = torch.ones(B * cols, dtype=torch.int32, device="cuda")
    mask[0] = 0
    assert m.attend(q2, ln, mask01=mask)[0].eq(0).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B, cols, S, heads, d", DEALT)
def test_what_lies_outside_the_window_is_not_looked_at_by_several_ctas(api, dtype, B, cols, S, heads, d):
    lens, offs = [S - 40, 70, 33][:B], [13, S - 70, 40][:B]
    m, q, ln, of, scale, out = attend_case(api, dtype, B, cols, S, heads, d, lens, offs)
    for b in range(B):
        for at in (slice(0, offs[b]), slice(offs[b] + lens[b], S)):
            m.codes[b, at] = 255
            m.scales[b, at] = float("nan")
    assert torch.equal(m.attend(q, ln, of, scale=scale), out)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_attend_with_large_and_small_queries(api, dtype):
    """Scores in the thousands (one slot takes all the weight), scores of nothing (equal weights), zero queries."""
    for mul in (30.0, 1e-6, 0.0) + (() if dtype == "f16" else (1e-30, 1e5)):
        attend_case(api, dtype, 2, 12, 77, 1, 256, [77, 50], [0, 5], seed=5, qmul=mul)
    attend_case(api, dtype, 2, 5, 600, 4, 64, [600, 1], [0, 599], seed=5, qmul=20.0, scale=-0.7)


@pytest.mark.parametrize("dtype, qmag, scale", [("f32", 3.0e38, 1.0), ("f32", 3.0e38, -1.0), ("f32", 1.0e38, 2.5), ("f32", 1.0, 3.0e38), ("f32", 2.0 ** -100, 2.0 ** 127), ("bf16", 3.0e38, 1.0), ("bf16", 1.0, -3.0e38), ("f16", 60000.0, 5.0e33), ("f16", 1.0, 3.0e38)])
@pytest.mark.parametrize("B, cols, S, heads, d", DEALT + OTHERS)
def test_attend_with_scores_at_the_end_of_the_range(api, dtype, qmag, scale, B, cols, S, heads, d):
    """Scores of up to some 2^126, from large queries or a large scale: the slots of the largest score share all the weight, by equal parts.  (One element of a
    query is not zero, so a score is one product, rounded; the memory's values differ by 2^-11 of themselves or not at all, so that the slots that share
    are those of the largest value.)"""
    g = gen(S + d)
    x = 0.25 * torch.rand(S, B, heads, -(-d // 32), 1, generator=g, device="cuda").expand(S, B, heads, -(-d // 32), 32).reshape(S, B, heads, -1)[..., :d]
    u = torch.where(torch.rand(S, B, heads, d, generator=g, device="cuda") < 0.5, -1.0, 1.0)
    m = api.memory4(B, S, d, heads=heads).pack((x * u).reshape(S, B, heads * d))
    q = torch.zeros(B * cols, heads, d, device="cuda")
    at = torch.randint(0, d, (B * cols, heads), generator=g, device="cuda")
    q.scatter_(2, at[..., None], torch.where(torch.rand(B * cols, heads, 1, generator=g, device="cuda") < 0.5, -qmag, qmag))
    q = q.to(ref.TYPES[dtype]).view(B * cols, heads * d)
    ln = torch.full((B,), S, dtype=torch.int32, device="cuda")
    out = m.attend(q, ln, scale=scale).double().view(B, cols, heads, d)
    v = m.unpack().double()
    z = torch.einsum("bchd,bshd->bchs", q.double().view(B, cols, heads, d), v) * scale
    best = (z == z.amax(-1, keepdim=True)).double()
    want = torch.einsum("bchs,bshd->bchd", best, v) / best.sum(-1, keepdim=True)
    tol = (sum_tol(S) + 4 * EPS) * 0.25 + ref.HALF_STEP[dtype] * want.abs()
    assert bool(((out - want).abs() <= tol).all())


@pytest.mark.parametrize("dtype, small", [("f32", 2.0 ** -28), ("bf16", 2.0 ** -30), ("f16", 2.0 ** -26)])
@pytest.mark.parametrize("B, cols, S, heads, d", DEALT + OTHERS)
def test_attend_with_queries_of_very_different_elements(api, dtype, small, B, cols, S, heads, d):
    """Elements far below their row's largest decide, where the memory is large: each counts with its type's precision."""
    g = gen(d)
    top = 32768.0 if dtype == "f16" else 1.0
    q = torch.randn(B * cols, heads, d, generator=g, device="cuda") * (small * top)
    q[..., :32] = top  # times memory values of up to 2e-6
    amp = torch.full((d,), 2.0 ** 12, device="cuda")
    amp[:32] = 2.0 ** -19
    v = torch.tanh(torch.randn(S, B, heads, d, generator=g, device="cuda")) * amp
    m = api.memory4(B, S, d, heads=heads).pack(v.view(S, B, heads * d))
    q = q.to(ref.TYPES[dtype]).view(B * cols, heads * d)
    ln = torch.full((B,), S, dtype=torch.int32, device="cuda")
    scale = 4.0 / (small * top * 2.0 ** 12 * d ** 0.5)
    out = m.attend(q, ln, scale=scale)
    check_attend(out, ref.unpack(m.codes.cpu().numpy(), m.scales.cpu().numpy(), d), f64(q), [S] * B, [0] * B, scale, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("cols, d, teams", [(3, 264, 0), (1200, 1000, 2), (1200, 264, 4), (1200, 100, 16)])
@pytest.mark.parametrize("peak", [0, 100001])
def test_attend_to_one_large_weight_and_a_long_flat_tail(api, dtype, cols, d, teams, peak):
    """One slot, and 2^19 others whose weights of 2^-25.5 of its are, together, 2^-6.5 of the whole.  1200 columns: the window is one CTA's, whose teams of
    warps have an equal share of the slots each; 3: it is shared by many.

    Tolerance.  out = v0 (1 - tail) / (1 + tail), since the others' values are the negative one's.  A score's error of t changes a tail weight by a factor 1 + t, out by
    2 tail t.  The team that has the large weight adds its share of the tail to it: in 16 bits by tensor-core additions of 16 slots, cut off (2 eps of the sums
    each), in 32 bits by additions of 32 slots, rounded (eps); numerator and denominator alike.  16-bit types have weights in steps of 2^-31 of the
    largest: half a step is 2^-6.5 of a tail weight.  A window that many share has none of that: their sums are added in a few hundred roundings."""
    S = 1 << 19
    assert (attend_ways(api, 1, cols, S, 1, d) == 0) == (teams > 0)
    g = gen(d)
    u = torch.where(torch.rand(d, generator=g, device="cuda") < 0.5, -0.5, 0.5)
    m = api.memory4(1, S, d)
    m.pack((-u).expand(S, 1, d))
    m.pack(u.expand(1, 1, d), slot0=peak)
    v = m.unpack(slot0=peak, S=1).double().view(d)
    q = (u * 2).to(ref.TYPES[dtype]).repeat(cols, 1)
    scale = 12.75 * np.log(2.0) / float((q[0].double() * v).sum())  # scores of +-12.75 log 2
    out = m.attend(q, torch.full((1,), S, dtype=torch.int32, device="cuda"), scale=scale).double()
    tail = (S - 1) * 2.0 ** -25.5
    want = v * ((1 - tail) / (1 + tail))
    share = S / teams if teams else 0
    cut = 2 * (share / 16 * 2 * EPS if dtype != "f32" else share / 32 * EPS) + 512 * EPS
    step = 2 * tail * (1 / teams if teams else 2.0 ** -6) * (2.0 ** -6.5 if dtype != "f32" else 2.0 ** -17.5)
    tol = float(v.abs().max()) * (2 * tail * 2 * sum_tol(d) * 13 + cut + step) + ref.HALF_STEP[dtype] * want.abs()
    err = (out - want).abs()
    assert bool((err <= tol).all()), (float(err.max()), float((err / tol).max()))


@pytest.mark.parametrize("B, cols, S, heads, d", DEALT + OTHERS)
def test_attend_in_fp16_is_rounded_once(api, B, cols, S, heads, d):
    """Beside the result's rounding to fp16 there are only those of 32 bits: few slots of comparable weights, where a weight's rounding to a half would show."""
    g = gen(7 * d)
    m = api.memory4(B, S, d, heads=heads).pack(torch.tanh(torch.randn(S, B, heads * d, generator=g, device="cuda")))
    q = (0.1 * torch.randn(B * cols, heads * d, generator=g, device="cuda")).half()
    v = ref.unpack(m.codes.cpu().numpy(), m.scales.cpu().numpy(), d)
    for n in (2, 3, 7):
        lens, offs = [n] * B, [(b * 17) % (S - n) for b in range(B)]
        out = m.attend(q, torch.tensor(lens, dtype=torch.int32, device="cuda"), torch.tensor(offs, dtype=torch.int32, device="cuda"), scale=d ** -0.5)
        want, mag = ref.attend(v, f64(q), lens, offs, d ** -0.5)
        tol = np.abs(v).max() * (2 * sum_tol(d) * mag + 4 * sum_tol(n))[..., None] + ref.HALF_STEP["f16"] * np.abs(want) + 2.0 ** -25  # (half a step of its subnormals)
        assert (np.abs(f64(out).reshape(want.shape) - want) <= tol).all()


def test_attend_on_strided_queries_and_outputs(api):
    g = gen(11)
    B, cols, S, d = 3, 4, 45, 100
    hs = torch.tanh(torch.randn(S, B, d, generator=g, device="cuda"))
    m = api.memory4(B, S, d).pack(hs)
    lens = torch.tensor([45, 20, 3], dtype=torch.int32, device="cuda")
    for t in ref.TYPES.values():
        wide = torch.randn(B * cols, d + 7, generator=g, device="cuda").to(t)
        q = wide[:, 3:3 + d]
        out = torch.full((B * cols, d + 5), 9.0, dtype=t, device="cuda")
        m.attend(q, lens, out=out[:, 2:2 + d])
        assert torch.equal(out[:, 2:2 + d], m.attend(q.contiguous(), lens)) and out[:, :2].eq(9).all() and out[:, 2 + d:].eq(9).all()


def test_attend_repeats_itself(api):
    """Equal inputs give equal bits, whatever ran before; and a sentence's result does not depend on the others."""
    m, q, ln, of, scale, out = attend_case(api, "f32", 4, 12, 2000, 1, 300, [2000, 1500, 1, 700], [0, 500, 3, 0])
    torch.randn(1 << 24, device="cuda")
    assert torch.equal(m.attend(q, ln, of, scale=scale), out)


def test_attend_at_the_far_end_of_a_long_memory(api):
    """More than 2^32 bytes of codes: offsets of 64 bits."""
    S, d = (1 << 23) + 1000, 1024
    if torch.cuda.mem_get_info()[0] < 8 << 30:
        pytest.skip("needs 8 GB")
    m = api.memory4(1, S, d)
    g = gen(2)
    hs = torch.tanh(torch.randn(45, 1, d, generator=g, device="cuda"))
    q = torch.tanh(torch.randn(5, d, generator=g, device="cuda"))
    m.pack(hs, slot0=S - 45)
    n, o = torch.tensor([45], dtype=torch.int32, device="cuda"), torch.tensor([S - 45], dtype=torch.int32, device="cuda")
    small = api.memory4(1, 45, d).pack(hs)
    assert torch.equal(m.unpack(slot0=S - 45, S=45), small.unpack())
    check_attend(m.attend(q, n, o), f64(small.unpack()), f64(q), [45], [0], 1.0, "f32")


# ------------------------------------------------------------------ linear
def linear_case(api, dtype, n, K, N, act="none", bias=True, residual=False, pad=(0, 0, 0, 0), seed=0, inplace=False, xmul=1.0):
    """pad: how much further apart than they are long the rows of W, X, R and Y are."""
    g = gen(seed)
    W = randn(g, n, K + pad[0], dtype=dtype)[:, :K]
    W.mul_(K ** -0.5)
    X = (xmul * randn(g, N, K + pad[1])).to(ref.TYPES[dtype])[:, :K]
    b = 0.5 * randn(g, n) if bias else None
    Y = torch.full((N, n + pad[3]), 7.0, dtype=ref.TYPES[dtype], device="cuda")
    R = randn(g, N, n + pad[2], dtype=dtype)[:, :n] if residual else None
    if inplace:
        Y[:, :n] = R
        want_R, R = R, Y[:, :n]
    else:
        want_R = R
    z = X.double() @ W.double().t()
    if bias:
        z = z + b.double()
    want = ref.act(z, act)
    if residual:
        want = want + want_R.double()
    out = api.linear(W, X, bias=b, act=act, residual=R, out=Y[:, :n])
    mag = X.double().abs() @ W.double().abs().t() + (b.double().abs() if bias else 0)
    # the activations' slopes are at most 1.13; they are evaluated to within a few roundings of 32 bits
    tol = 1.13 * sum_tol(K) * mag + 16 * EPS * (1 + want.abs()) + ref.HALF_STEP[dtype] * (want.abs() + 1e-7)
    err = (out.double() - want).abs()
    assert bool((err <= tol).all()), (float(err.max()), float((err / tol).max()))
    assert Y[:, n:].eq(7).all()
    return W, X, b, out


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n, K, N", [
    (1, 1, 1), (3, 5, 2), (64, 64, 1), (1000, 2000, 12), (1000, 2000, 5), (129, 257, 16), (200, 1000, 17), (500, 96, 33), (256, 512, 64), (300, 40, 65), (1000, 1000, 100),
    (1000, 2000, 768), (333, 777, 200), (777, 1024, 129), (2048, 320, 300), (130, 4096, 257), (37, 1173, 1), (4100, 64, 513), (515, 8, 1000), (8, 515, 1000), (300, 1, 300), (300, 3, 200), (245, 7428, 3), (40, 16384, 16), (100, 9001, 30), (512, 8192, 512), (1000, 2000, 64)])
def test_linear(api, dtype, n, K, N):
    linear_case(api, dtype, n, K, N, seed=n + K)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("act", ["none", "tanh", "sigmoid", "relu", "gelu", "silu"])
@pytest.mark.parametrize("n, K, N", [(200, 96, 7), (260, 160, 300)])
def test_linear_epilogues(api, dtype, act, n, K, N):
    linear_case(api, dtype, n, K, N, act, bias=False, seed=1)
    linear_case(api, dtype, n, K, N, act, residual=True, seed=2, xmul=4.0)
    linear_case(api, dtype, n, K, N, act, residual=True, inplace=True, seed=3)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("pad", [(8, 0, 0, 0), (0, 8, 24, 8), (3, 0, 0, 0), (0, 1, 0, 0), (5, 3, 1, 7), (4, 4, 4, 4)])
@pytest.mark.parametrize("n, K, N", [(136, 200, 9), (264, 136, 301), (141, 205, 40)])
def test_linear_strides(api, dtype, pad, n, K, N):
    linear_case(api, dtype, n, K, N, "tanh", residual=True, pad=pad, seed=4)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_linear_on_operands_that_start_anywhere(api, dtype):
    g = gen(8)
    t = ref.TYPES[dtype]
    for n, K, N in ((130, 96, 6), (270, 128, 200)):
        for off in (1, 2, 4, 8):
            Wb, Xb = randn(g, n * K + 16, dtype=dtype), randn(g, N * K + 16, dtype=dtype)
            W, X = Wb[off:off + n * K].view(n, K), Xb[16 - off:16 - off + N * K].view(N, K)
            out = torch.empty(N * n + 16, dtype=t, device="cuda")[off:off + N * n].view(N, n)
            api.linear(W, X, out=out)
            want, mag = X.double() @ W.double().t(), X.double().abs() @ W.double().abs().t()
            assert bool(((out.double() - want).abs() <= sum_tol(K) * mag + ref.HALF_STEP[dtype] * want.abs()).all())


def test_linear_in_32_bits_of_wide_ranges(api):
    """fp32 operands over the whole range of magnitudes that 3xTF32 must carry: nothing is rounded to half precision on the way."""
    g = gen(9)
    for n, K, N in ((100, 300, 5), (300, 300, 200)):
        W = randn(g, n, K) * torch.exp2(torch.randint(-60, 60, (n, 1), generator=g, device="cuda").float())
        X = randn(g, N, K) * torch.exp2(torch.randint(-40, 60, (N, 1), generator=g, device="cuda").float())
        out = api.linear(W, X).double()
        want, mag = X.double() @ W.double().t(), X.double().abs() @ W.double().abs().t()
        assert bool(((out - want).abs() <= sum_tol(K) * mag).all())


@pytest.mark.parametrize("N", [6, 3000])  # the kernel for few columns, the one on tcgen05
@pytest.mark.parametrize("K", [8, 32, 128, 512, 2000])
def test_linear_in_32_bits_beside_a_plain_product(api, N, K):
    """Errors of single operands' splitting, which a sum's tolerance hides: the root of the mean square and the mean, signed error, of results relative to the root of the
    sum of the products' squares (random signs) or to the result (positive operands), and next to a product in ordinary 32-bit arithmetic, step by step.

    Bounds.  An operand's hi + lo is off by 2^-22 at most, 0.8e-7 on the average and to either side; what a product leaves out, lo lo, is 0.8e-7 on the average
    and has no side: 1.2e-7 together, 2^-22 with a factor of two in hand, and a mean of 2^-24.  A tensor-core instruction cuts a sum off, by 2^-23 of what there is
    of it at most: of m of them in a row, (m + 1) / 2 times that.  The additions in 32 bits: 2^-23.  Operands just below 1 + 2^-10 all have the same hi and lo as
    large as it gets: off by 2^-22, all to one side."""
    g = gen(K + N)
    n = 1000
    m = min(16, -(-K // 8)) if N > 100 else min(8, 2 * -(-K // 128))
    cut = (m + 1) / 2 * 2.0 ** -23
    u = lambda *s: torch.rand(s, generator=g, device="cuda")  # noqa: E731
    below = lambda *s: 1 + 2.0 ** -10 - 2.0 ** -23 * torch.randint(1, 9, s, generator=g, device="cuda").float()  # noqa: E731
    for kind, make, one_side in (("signs", lambda *s: randn(g, *s), 2.0 ** -24), ("positive", lambda *s: 1 + u(*s), 2.0 ** -24), ("below", below, 2.0 ** -22 + 2.0 ** -24)):
        W, X = make(n, K), make(N, K)
        want = X.double() @ W.double().t()
        scale = want.abs() if kind != "signs" else ((X.double() ** 2) @ (W.double() ** 2).t()).sqrt()
        plain = torch.zeros(N, n, device="cuda")
        for k in range(K):
            plain += X[:, k:k + 1] * W[:, k]
        err, ours = [(y.double() - want) * want.sign() / scale for y in (plain, api.linear(W, X))]
        mean, rms = float(ours.mean()), float(ours.square().mean().sqrt())
        of_plain = float(err.mean()), float(err.square().mean().sqrt())
        assert abs(mean) <= one_side + cut, (kind, mean, rms, of_plain)
        assert rms <= 2.0 ** -22 + cut + 2.0 ** -23 + (one_side if kind == "below" else 0), (kind, mean, rms, of_plain)
        if kind == "signs" and K >= 512:  # (a plain sum's errors grow with its length)
            assert rms <= 2 * of_plain[1], (rms, of_plain)


@pytest.mark.parametrize("N", [6, 300])
def test_linear_in_32_bits_of_the_largest_numbers(api, N):
    """Operands next to the largest number do not round to an infinity on the way."""
    g = gen(N)
    top = torch.tensor([0x7f7fffff, 0x7f7ff000, 0x7f7fefff, 0x7f7fe000], dtype=torch.int32).view(torch.float32).cuda()
    W = (2.0 ** -20 * torch.rand(200, 64, generator=g, device="cuda"))
    X = torch.zeros(N, 64, device="cuda")
    X[:, 5] = top[torch.arange(N, device="cuda") % 4]
    X[1::2] *= -1
    for a, b in ((W, X), (X, W)):
        want = b.double() @ a.double().t()
        out = api.linear(a, b)
        assert bool(((out.double() - want).abs() <= sum_tol(64) * want.abs()).all())


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("N", [6, 200])
def test_linear_numbers_that_are_not_finite(api, dtype, N):
    """An infinity or a NaN in a column of X reaches that column alone, one in a row of W that output alone."""
    g = gen(10)
    n, K = 200, 130
    W, X = randn(g, n, K, dtype=dtype), randn(g, N, K, dtype=dtype)
    clean = api.linear(W, X, act="tanh")
    X2, W2 = X.clone(), W.clone()
    X2[3, 129] = float("nan")
    X2[4, 0] = float("inf")
    W2[150, 7] = float("nan")
    got = api.linear(W2, X2, act="tanh")
    assert got[3].isnan().all() and got[:, 150].isnan().all()
    keep_c = [c for c in range(N) if c not in (3, 4)]
    keep_n = [i for i in range(n) if i != 150]
    assert torch.equal(got[keep_c][:, keep_n], clean[keep_c][:, keep_n])
    # (3xTF32 splits an infinity into inf + NaN: the column is not finite, as inf * x is not)
    assert bool((got[4, keep_n].isnan() | (got[4, keep_n].abs() == 1)).all())


def test_linear_output_beyond_2_to_the_32(api):
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    n, N, K = 70000, 66000, 8
    g = gen(12)
    W, X = randn(g, n, K, dtype="bf16"), randn(g, N, K, dtype="bf16")
    out = api.linear(W, X)
    at = torch.tensor([0, 1, 31000, 61356, 61357, 65535, 65999], device="cuda")
    want = X[at].double() @ W.double().t()
    mag = X[at].double().abs() @ W.double().abs().t()
    assert bool(((out[at].double() - want).abs() <= sum_tol(K) * mag + ref.HALF_STEP["bf16"] * want.abs()).all())


# ------------------------------------------------------------------ selection
def select_case(api, z, scores, beam, k, lse=None, done=None, eos=1):
    got = api.beam_select(z, scores, beam, k, lse=lse, done=done, eos=eos)
    c = lambda t: None if t is None else t.cpu().numpy()  # noqa: E731
    want = ref.select(z.float().cpu().numpy(), c(scores), beam, k, c(lse), c(done), eos)
    for a, b, name in zip(got, want, ("values", "words", "parents")):
        np.testing.assert_array_equal(a.cpu().numpy(), b, err_msg=name)
    return got


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n, beam, V, k", [
    (1, 1, 1, 1), (1, 1, 7, 7), (2, 3, 5, 15), (1, 12, 40000, 12), (5, 12, 5003, 12), (3, 5, 129, 64), (7, 2, 1000, 4), (40, 8, 3001, 8), (2, 32, 20001, 64), (1, 1, 200000, 33),
    (300, 4, 777, 5), (2, 64, 33, 64), (1, 7, 100003, 50)])
def test_beam_select(api, dtype, n, beam, V, k):
    g = gen(n + V)
    z = 2 * randn(g, n * beam, V, dtype=dtype)
    scores = -20 + 3 * randn(g, n * beam)
    lse = torch.logsumexp(z.float(), 1)
    select_case(api, z, scores, beam, k, lse=lse)
    select_case(api, z, scores, beam, k)


@pytest.mark.parametrize("dtype, n, beam, V", [("f32", 1, 32, 200001), ("f32", 2, 25, 190003), ("bf16", 1, 50, 200000), ("f16", 1, 3, 3000001)])
def test_beam_select_of_sentences_too_long_for_a_cluster(api, dtype, n, beam, V):
    """Lists of many CTAs, merged by a second launch: in shared memory, out of it, and with more ties than it ranks."""
    g = gen(V)
    z = 2 * randn(g, n * beam, V, dtype=dtype)
    scores = -20 + 3 * randn(g, n * beam)
    done = (torch.rand(n * beam, generator=g, device="cuda") < 0.3).int()
    for k in (1, 8, 64):
        select_case(api, z, scores, beam, k)
    select_case(api, z, scores, beam, 12, done=done, eos=V - 1)
    z.zero_()
    for k in (8, 64):
        _, word, parent = select_case(api, z, torch.zeros_like(scores), beam, k)
        assert word[0].tolist() == list(range(k)) and parent[0].eq(0).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n, beam, V", [(3, 12, 2001), (2, 5, 30000), (1, 12, 120000)])
def test_beam_select_finished_and_dead_hypotheses(api, dtype, n, beam, V):
    g = gen(V)
    z = 2 * randn(g, n * beam, V, dtype=dtype)
    scores = -20 + 3 * randn(g, n * beam)
    done = (torch.rand(n * beam, generator=g, device="cuda") < 0.4).int()
    scores[2] = float("-inf")
    scores[beam - 1] = float("nan")
    z[1, 5] = float("nan")
    z[1, 9:40] = float("-inf")
    lse = torch.logsumexp(torch.nan_to_num(z.float(), nan=0.0), 1)
    for eos in (1, 0, V - 1):
        select_case(api, z, scores, beam, beam, lse=lse, done=done, eos=eos)
    # every hypothesis finished: as many candidates as hypotheses, the rest of the output is empty
    k = min(64, beam + 3)
    scores = -20 + 3 * randn(g, n * beam)
    val, word, parent = select_case(api, z, scores, beam, k, done=torch.ones_like(done), eos=2)
    assert word[:, :beam].eq(2).all() and word[:, beam:].eq(-1).all() and parent[:, beam:].eq(-1).all() and val[:, beam:].eq(float("-inf")).all()
    # no hypothesis alive
    val, word, parent = select_case(api, z, torch.full_like(scores, float("-inf")), beam, 4)
    assert word.eq(-1).all() and parent.eq(-1).all()
    done[:] = torch.arange(n * beam, device="cuda") % 3
    val, word, parent = select_case(api, torch.full_like(z, float("-inf")), scores, beam, 8, done=done)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("V", [50, 5000, 70001])
def test_beam_select_ties_go_to_the_lowest_candidate(api, dtype, V):
    """All candidates equal; a few values only; +0 and -0; +inf."""
    n, beam, k = 2, 6, 20
    z = torch.zeros(n * beam, V, dtype=ref.TYPES[dtype], device="cuda")
    s = torch.zeros(n * beam, device="cuda")
    _, word, parent = select_case(api, z, s, beam, k)
    assert word[0].tolist() == list(range(k)) and parent[1].tolist() == [beam] * k
    g = gen(4)
    z = torch.randint(-2, 2, (n * beam, V), generator=g, device="cuda").to(ref.TYPES[dtype])
    z = torch.where(z == 1, -0.0, z.float()).to(ref.TYPES[dtype])
    select_case(api, z, s, beam, 64)
    select_case(api, z, -s, beam, 64)
    z[3, V // 2] = z[1, V - 1] = float("inf")
    select_case(api, z, s, beam, k)
    up = torch.arange(V, device="cuda").float().repeat(n * beam, 1).to(ref.TYPES[dtype])  # every new value is better than all before
    select_case(api, up, s, beam, 64)
    select_case(api, -up, s, beam, 64)


@pytest.mark.parametrize("n, beam, V, k", [(1, 12, 40000, 12), (3, 1, 300, 1), (64, 12, 4000, 12), (20, 2, 64, 5)])
def test_beam_select_of_one_outstanding_candidate_per_segment(api, n, beam, V, k):
    """A segment that went missing shows: the best candidates lie one to a segment, in other segments in every call, right after launches that
    leave the multiprocessors' shared memory full of larger numbers."""
    g = gen(V + 1)
    scores = torch.zeros(n * beam, device="cuda")
    junk = 1e6 + torch.rand(n * beam, V, generator=g, device="cuda")
    low = -100 - torch.rand(n * beam, V, generator=g, device="cuda")
    zs, wants = [], []
    for i in range(30):
        z = low.clone().view(n, beam * V)
        at = torch.stack([torch.randperm((beam * V + 127) // 128, generator=g, device="cuda")[:k] for _ in range(n)])
        at = (128 * at + torch.randint(0, 128, at.shape, generator=g, device="cuda")).clamp(max=beam * V - 1)
        best = torch.rand(n, at.shape[1], generator=g, device="cuda") + torch.arange(at.shape[1], device="cuda")
        z.scatter_(1, at, best)
        zs.append(z.view(n * beam, V))
        val, cand = z.sort(1, descending=True)
        wants.append((val[:, :at.shape[1]], cand[:, :at.shape[1]]))
    for z, (val, cand) in zip(zs, wants):
        api.beam_select(junk, scores, beam, k)
        got, word, parent = api.beam_select(z, scores, beam, k)
        m = val.shape[1]
        first = torch.arange(n, device="cuda")[:, None] * beam
        assert torch.equal(got[:, :m], val) and torch.equal((parent[:, :m].long() - first) * V + word[:, :m], cand)


@pytest.mark.parametrize("beam, V, k", [(5_100_000, 2, 1), (5_050_000, 1, 1), (600_000, 2, 64)])
def test_beam_select_of_millions_of_hypotheses(api, beam, V, k):
    """A segment per row: thousands of lists to merge."""
    g = gen(beam)
    z, scores = randn(g, beam, V), -20 + 3 * randn(g, beam)
    val, word, parent = api.beam_select(z, scores, beam, k)
    cand = (scores[:, None] + z).view(-1)
    want, at = torch.sort(cand, descending=True, stable=True)
    assert torch.equal(val[0], want[:k]) and torch.equal(parent[0].long() * V + word[0], at[:k])


def test_beam_select_on_rows_that_start_anywhere(api):
    g = gen(6)
    for dtype in ref.TYPES:
        for V, ld in ((1001, 1003), (999, 1000), (4097, 4097), (64, 65)):
            buf = randn(g, 3 * 4 * ld + 8, dtype=dtype)
            for off in (0, 1, 3):
                z = buf[off:off + 12 * ld].view(12, ld)[:, :V]
                select_case(api, z, randn(g, 12), 4, 6)


# ------------------------------------------------------------------ reorder
@pytest.mark.parametrize("n_src, n, dtype, widths", [
    (12, 12, torch.float32, (1000, 1000, 64)), (24, 60, torch.bfloat16, (333,)), (7, 5, torch.uint8, (1, 3, 17)), (768, 768, torch.float32, (1000,) * 5), (4, 1, torch.float16, (6, 2)),
    (1, 9, torch.float32, (130,))])
def test_beam_reorder(api, n_src, n, dtype, widths):
    g = gen(n)
    xs = [(100 * torch.randn(n_src, w, generator=g, device="cuda")).to(dtype) for w in widths]
    p = torch.randint(-1, n_src, (n,), generator=g, device="cuda", dtype=torch.int32)
    out = api.beam_reorder(xs, p)
    for x, o in zip(xs, out):
        want = torch.where((p >= 0)[:, None], x[p.clamp(min=0).long()], torch.zeros((), dtype=dtype, device="cuda"))
        assert torch.equal(o, want)


@pytest.mark.parametrize("beam", [1, 2, 5, 12, 16, 33, 64])
def test_beam_reorder_in_place(api, beam):
    g = gen(beam)
    n = 6 * beam
    xs = [torch.randn(n, w, generator=g, device="cuda") for w in (1000, 3, 40)] + [torch.randn(n, 33, generator=g, device="cuda").half()]
    p = torch.randint(0, beam, (6, beam), generator=g, device="cuda", dtype=torch.int32) + torch.arange(6, device="cuda", dtype=torch.int32)[:, None] * beam
    p.view(-1)[n // 2] = -1
    want = [torch.where((p.view(-1) >= 0)[:, None], x[p.view(-1).clamp(min=0).long()], 0.0) for x in xs]
    other = torch.empty_like(xs[1])
    got = api.beam_reorder(xs + [xs[1].clone()], p, out=xs + [other], group=beam)  # the last one out of place
    for a, b in zip(got, want + [want[1]]):
        assert torch.equal(a, b)


def test_beam_reorder_reports_a_parent_that_is_no_column(api):
    assert api.lib().zrnn_tc_error() == 0
    x = torch.randn(6, 100, device="cuda")
    keep = x.clone()
    p = torch.tensor([0, 6, 2, 2**31 - 1, -7, 1], dtype=torch.int32, device="cuda")
    out, = api.beam_reorder([x], p)
    torch.cuda.synchronize()
    assert api.lib().zrnn_tc_error() == 101
    assert out[[1, 3, 4]].eq(0).all() and torch.equal(out[[0, 2, 5]], x[[0, 2, 1]])
    api.beam_reorder([x], torch.tensor([1, 0, 3, 2, 3, 4], dtype=torch.int32, device="cuda"), out=[x], group=3)
    torch.cuda.synchronize()
    assert api.lib().zrnn_tc_error() == 101  # columns 2 and 4 asked for the other group
    assert torch.equal(x, keep[[1, 0, 2, 3, 3, 4]])


# ------------------------------------------------------------------ together
class Step:
    """A decoder's step made of the operators: attention over the packed source, the combiner, the vocabulary's logits, selection, reorder."""

    def __init__(self, api, n=3, beam=4, H=96, V=501, S=37, dtype="f32"):
        g = gen(21)
        t = ref.TYPES[dtype]
        self.api, self.n, self.beam, self.H, self.V, self.dtype = api, n, beam, H, V, dtype
        self.hs = torch.tanh(torch.randn(S, n, H, generator=g, device="cuda")).to(t)
        self.lens = torch.tensor([S, 9, 1][:n], dtype=torch.int32, device="cuda")
        self.offs = S - self.lens
        self.Wc = (torch.randn(H, 2 * H, generator=g, device="cuda") * 0.2).to(t)
        self.bc = torch.randn(H, generator=g, device="cuda") * 0.1
        self.D = torch.randn(V, H, generator=g, device="cuda").to(t)
        self.bd = torch.randn(V, generator=g, device="cuda") * 0.1
        self.h = torch.tanh(torch.randn(n * beam, H, generator=g, device="cuda")).to(t)
        self.scores = torch.randn(n * beam, generator=g, device="cuda") - 3

    def run(self, mem):
        a = self.api
        ctx = mem.attend(self.h, self.lens, self.offs)
        ht = a.linear(self.Wc, torch.cat([ctx, self.h], 1), bias=self.bc, act="tanh", residual=self.h)
        z = a.linear(self.D, ht, bias=self.bd)
        lse = torch.logsumexp(z.float(), 1)
        val, word, parent = a.beam_select(z, self.scores, self.beam, self.beam, lse=lse)
        new, = a.beam_reorder([ht], parent)
        return ctx, ht, z, lse, val, word, parent, new

    def check(self, mem, got):
        ctx, ht, z, lse, val, word, parent, new = got
        v = ref.unpack(mem.codes.cpu().numpy(), mem.scales.cpu().numpy(), self.H)
        check_attend(ctx, v, f64(self.h), self.lens.tolist(), self.offs.tolist(), 1.0, self.dtype)
        X = torch.cat([ctx, self.h], 1).double()
        want = torch.tanh(X @ self.Wc.double().t() + self.bc.double()) + self.h.double()
        tol = sum_tol(2 * self.H) * (X.abs() @ self.Wc.double().abs().t() + 1) + (16 * EPS + ref.HALF_STEP[self.dtype]) * (1 + want.abs())
        assert bool(((ht.double() - want).abs() <= tol).all())
        want = ht.double() @ self.D.double().t() + self.bd.double()
        tol = sum_tol(self.H) * (ht.double().abs() @ self.D.double().abs().t() + 1) + (16 * EPS + ref.HALF_STEP[self.dtype]) * (1 + want.abs())
        assert bool(((z.double() - want).abs() <= tol).all())
        w = ref.select(z.float().cpu().numpy(), self.scores.cpu().numpy(), self.beam, self.beam, lse.cpu().numpy())
        for a, b in zip((val, word, parent), w):
            np.testing.assert_array_equal(a.cpu().numpy(), b)
        assert torch.equal(new, ht[parent.view(-1).long()])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_a_step_of_all_operators(api, dtype):
    s = Step(api, dtype=dtype)
    mem = api.memory4(3, 37, 96).pack(s.hs)
    s.check(mem, s.run(mem))


def test_a_captured_step_gives_what_the_calls_give(api):
    """Capture, replay on changed inputs, two graphs replayed on two streams at once."""
    steps = [Step(api), Step(api, n=2, beam=12, H=320, V=3000)]
    mems = [api.memory4(s.n, 37, s.H).pack(s.hs) for s in steps]
    graphs, outs = [], []
    for s, m in zip(steps, mems):
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            s.run(m)
        torch.cuda.current_stream().wait_stream(st)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(s.run(m))
        graphs.append(gr)
    for round_ in range(3):
        for s in steps:
            s.h.copy_(torch.tanh(torch.randn(s.h.shape, generator=gen(50 + round_), device="cuda")))
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for _ in range(5):
            for gr, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    gr.replay()
        torch.cuda.synchronize()
        for s, m, o in zip(steps, mems, outs):
            s.check(m, o)
            for a, b in zip(o, s.run(m)):
                assert torch.equal(a, b)


def test_calls_on_two_streams_at_once(api):
    """Each call's scratch memory is its own."""
    m, q, ln, of, scale, out = attend_case(api, "f32", 2, 12, 5000, 1, 256, [5000, 4000], [0, 1000])
    g = gen(31)
    z, sc = 2 * randn(g, 24, 60000), randn(g, 24)
    W, X = randn(g, 700, 333), randn(g, 300, 333)
    base = [out, *api.beam_select(z, sc, 12, 12), api.linear(W, X)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(6):
        for st in streams:
            with torch.cuda.stream(st):
                got.append([m.attend(q, ln, of, scale=scale), *api.beam_select(z, sc, 12, 12), api.linear(W, X)])
    torch.cuda.synchronize()
    for r in got:
        for a, b in zip(r, base):
            assert torch.equal(a, b)


def test_the_calls_allocate_nothing(api):
    """Through the C ABI, with the caller's workspaces."""
    s = Step(api)
    mem = api.memory4(3, 37, 96).pack(s.hs)
    s.run(mem)
    torch.cuda.synchronize()
    before = torch.cuda.mem_get_info()[0]
    for _ in range(10):
        s.run(mem)
    torch.cuda.synchronize()
    assert torch.cuda.mem_get_info()[0] >= before


def test_the_c_abi_allocates_nothing(api):
    """Every call with the caller's buffers and workspaces, at sizes that need one: neither torch's allocator nor the device's free memory moves, from the
    second call of a size on and for larger ones after it (the first loads the kernels)."""
    L = api.lib()

    def step(scale, run):
        S, n, K, N, V = 4000 * scale, 512 * scale, 333, 512 * scale, 190003 * scale
        f32 = dict(dtype=torch.float32, device="cuda")
        t = dict(x=torch.zeros(S, 2, 64, **f32), q=torch.zeros(6, 64, **f32), ctx=torch.empty(6, 64, **f32), back=torch.empty(2, S, 64, **f32), W=torch.zeros(n * 8, K, **f32), X=torch.zeros(N * 4, K, **f32),
                 Y=torch.empty(N * 4, n * 8, **f32), z=torch.zeros(25, V, **f32), s=torch.zeros(25, **f32), val=torch.empty(12, **f32), moved=torch.empty(12, 100, **f32), state=torch.zeros(25, 100, **f32),
                 codes=torch.empty(2, S, 1, 32, dtype=torch.uint8, device="cuda"), scales=torch.empty(2, S, 1, 2, dtype=torch.float16, device="cuda"), lens=torch.full((2,), S, dtype=torch.int32, device="cuda"),
                 word=torch.empty(12, dtype=torch.int32, device="cuda"), parent=torch.empty(12, dtype=torch.int32, device="cuda"))
        p = {k: v.data_ptr() for k, v in t.items()}
        sizes = [ctypes.c_size_t() for _ in range(3)]
        assert L.zrnn_memory4_attend_workspace(2, 3, S, 1, 64, ctypes.byref(sizes[0])) == 0
        assert L.zrnn_linear_workspace(0, n * 8, N * 4, K, p["W"], K, p["X"], K, ctypes.byref(sizes[1])) == 0
        assert L.zrnn_beam_select_workspace(0, 1, 25, V, 12, ctypes.byref(sizes[2])) == 0
        assert all(z.value > 0 for z in sizes)
        work = [torch.empty(z.value, dtype=torch.uint8, device="cuda") for z in sizes]
        st = torch.cuda.current_stream().cuda_stream

        def calls():
            one = lambda a: (ctypes.c_void_p * 1)(a)  # noqa: E731
            assert [L.zrnn_memory4_pack(0, p["x"], 128, 64, S, 2, 1, 64, 0, S, p["codes"], p["scales"], st),
                    L.zrnn_memory4_unpack(0, p["codes"], p["scales"], 2, S, 1, 64, 0, S, p["back"], st),
                    L.zrnn_memory4_attend(0, p["codes"], p["scales"], 2, S, 1, 64, p["lens"], None, p["q"], 64, 3, None, 1.0, p["ctx"], 64, work[0].data_ptr(), sizes[0].value, st),
                    L.zrnn_linear(0, 1, n * 8, N * 4, K, p["W"], K, p["X"], K, None, None, 0, p["Y"], n * 8, work[1].data_ptr(), sizes[1].value, st),
                    L.zrnn_beam_select(0, p["z"], V, None, p["s"], None, 1, 25, V, 12, 1, p["val"], p["word"], p["parent"], work[2].data_ptr(), sizes[2].value, st),
                    L.zrnn_beam_reorder(1, one(p["state"]), one(p["moved"]), (ctypes.c_size_t * 1)(400), p["parent"], 12, 25, 1, st)] == [0] * 6
        if run:
            calls()
            torch.cuda.synchronize()
        return t, work, calls

    keep = step(1, True)
    larger = step(2, False)
    torch.cuda.synchronize()
    before = torch.cuda.mem_get_info()[0], torch.cuda.memory_stats()["allocation.all.allocated"]
    for calls in (keep[2], larger[2]) * 3:
        calls()
    torch.cuda.synchronize()
    assert (torch.cuda.mem_get_info()[0], torch.cuda.memory_stats()["allocation.all.allocated"]) == before
    assert L.zrnn_tc_error() == 0


@pytest.mark.parametrize("dtype", [3, 0, 1, 4])  # exact fp32, fp16 split, bf16, 3xTF32
@pytest.mark.parametrize("H, S, B, cols", [(64, 20, 3, 1), (320, 50, 5, 12), (1000, 33, 2, 4)])
def test_attention_layer_over_a_source_in_4_bits(api, dtype, H, S, B, cols):
    """The layer gives what it gives over the same numbers in 32 bits: the two contexts differ by roundings of 32 bits (sums over S and H
    products), which the combiner's sum of 2 H products and tanh pass on; with bf16 operands a rounding may fall to the other side."""
    g = gen(H)
    rng = np.random.default_rng(H)
    att = api.attention_layer(H, 10, att_type=api.ATT_GLOBAL_DOT, dtype=dtype)
    w = [rng.uniform(-0.1, 0.1, n).astype(np.float32) for n in (H * H, H * H, H, H, H * H, H * H)]
    att.load_weights(w)
    hs = torch.tanh(0.5 * torch.randn(S, B, H, generator=g, device="cuda"))
    lens = torch.tensor([S, S // 2, 3, 1, S - 1][:B], dtype=torch.int32, device="cuda")
    offs = S - lens
    m = api.memory4(B, S, H).pack(hs)
    values = m.unpack().view(B, S, H).permute(1, 0, 2).contiguous()
    h = torch.tanh(0.3 * torch.randn(B * cols, H, generator=g, device="cuda")).view(-1)
    mask = torch.ones(B * cols, dtype=torch.int32, device="cuda")
    mask[-1] = 0
    att.prep_minibatch_info(values.view(-1), S, B, lens, offs, cols_per_sentence=cols)
    want = att.forward_prop(h, mask)
    att.prep_minibatch_memory4(m, lens, offs, cols_per_sentence=cols)
    got = att.forward_prop(h, mask)
    # the context's error times the row sums of |W_c1| (0.05 H), and for bf16 a step of 2^-8 of a context of up to 1 with random signs
    tol = 0.05 * H * 2 * sum_tol(H) if dtype != 1 else 0.06 * H ** 0.5 * 2.0 ** -8 + 2.0 ** -10
    assert float((got - want).abs().max()) <= tol
    assert got.view(B * cols, H)[-1].eq(0).all()
    with pytest.raises(api.ZrnnError):
        att.forward_prop(h, mask, want_alignments=True)
    with pytest.raises(api.ZrnnError):
        att.forward_prop_viterbi(h, mask)
    if cols > 1:
        with pytest.raises(api.ZrnnError):
            att.forward_prop(h[: (cols + 1) * H].contiguous(), mask[: cols + 1].contiguous())
    att.prep_minibatch_info(values.view(-1), S, B, lens, offs, cols_per_sentence=cols)
    assert torch.equal(att.forward_prop(h, mask), want)
    local = api.attention_layer(H, 10, att_type=api.ATT_LOCAL_P, dtype=dtype)
    with pytest.raises(api.ZrnnError):
        local.prep_minibatch_memory4(m, lens, offs)


def test_the_first_calls_of_a_process_may_be_captured():
    """Nothing is set up by a call that a capture would not allow."""
    import os
    import subprocess
    import sys
    code = """
import torch
from zoph_rnn_b200 import api
torch.manual_seed(0)
r = lambda *s: torch.randn(*s, device="cuda")
hs, q, lens = torch.tanh(r(700, 2, 64)), r(6, 64), torch.tensor([700, 20], dtype=torch.int32, device="cuda")
W, X, X2, z, sc = r(300, 700), r(200, 700), r(3, 700), r(8, 40000), r(8)
m = api.memory4(2, 700, 64)
torch.cuda.synchronize()
def step():
    m.pack(hs)
    a = m.attend(q, lens)
    v, w, p = api.beam_select(z, sc, 4, 4)
    s, = api.beam_reorder([z], p)
    return a, api.linear(W, X, act="gelu"), api.linear(W, X2), api.linear(W.half(), X.half()), v, w, p, s
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    out = step()
g.replay()
torch.cuda.synchronize()
for a, b in zip(out, step()):
    assert torch.equal(a, b)
assert api.lib().zrnn_tc_error() == 0
print("captured")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    p = subprocess.run([sys.executable, "-c", code], cwd=root, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=300)
    assert p.returncode == 0 and "captured" in p.stdout, p.stdout


def test_several_threads_at_once(api):
    """The calls have no handle: threads call them side by side, each on its stream."""
    import threading
    s = [Step(api, n=2, beam=4 + i, H=64 * (i + 1), V=700 + i, dtype=d) for i, d in enumerate(("f32", "bf16", "f16", "f32"))]
    mem = [api.memory4(x.n, 37, x.H).pack(x.hs) for x in s]
    want = [x.run(m) for x, m in zip(s, mem)]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            for _ in range(20):
                got = s[i].run(mem[i])
                st.synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    bad.append(i)
    ts = [threading.Thread(target=work, args=(i,)) for i in range(len(s))]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not bad


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("n, K, N", [(520, 1024, 300), (1000, 520, 2000), (4100, 640, 5000)])
def test_linear_long_products_with_a_residual(api, dtype, n, K, N):
    """Several tiles per CTA, tiles that end in the middle, outputs as whole tiles and (odd rows) by stores; in place, too."""
    linear_case(api, dtype, n, K, N, "gelu", residual=True, seed=5)
    linear_case(api, dtype, n, K, N, "none", residual=True, inplace=True, seed=6)
    linear_case(api, dtype, n, K, N, "silu", residual=True, pad=(8, 16, 24, 8), seed=7)
    linear_case(api, dtype, n, K, N, "relu", residual=True, pad=(0, 0, 1, 3), seed=8)


@pytest.mark.parametrize("N", [32, 64, 96, 200])
def test_linear_in_32_bits_with_weights_from_far_memory(api, N):
    """One tile per multiprocessor, weights beyond the L2's size that come out of order: every call gives the same, and what it should."""
    g = gen(N)
    n, K = 18944, 2048
    W = [randn(g, n, K) * K ** -0.5 for _ in range(2)]
    X = randn(g, N, K)
    want = [X.double() @ w.double().t() for w in W]
    mag = [X.double().abs() @ w.double().abs().t() for w in W]
    first = [api.linear(w, X) for w in W]
    for a, b, m in zip(first, want, mag):
        assert bool(((a.double() - b).abs() <= sum_tol(K) * m).all())
    for _ in range(20):
        for w, a in zip(W, first):
            assert torch.equal(api.linear(w, X), a)


def test_many_sentences(api):
    """More sentences than a grid's dimension holds."""
    g = gen(40)
    z = randn(g, 70000, 9)
    select_case(api, z, randn(g, 70000), 1, 3)
    x = randn(g, 140000, 3)
    p = torch.arange(140000, device="cuda", dtype=torch.int32).flip(0).contiguous()
    out, = api.beam_reorder([x], p)
    assert torch.equal(out, x.flip(0))
    hs, q = torch.tanh(randn(g, 2, 70000, 32)), randn(g, 70000, 32)
    m = api.memory4(70000, 2, 32).pack(hs)
    lens = torch.randint(0, 3, (70000,), generator=g, device="cuda", dtype=torch.int32)
    out = m.attend(q, lens)
    at = [0, 1, 65534, 65535, 65536, 69999]
    v = f64(m.unpack())[at]
    check_attend(out[at], v, f64(q)[at], lens.cpu().numpy()[at], [0] * 6, 1.0, "f32")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_operands_and_outputs_side_by_side_in_one_matrix(api, dtype):
    """[context; state] without a copy: the attention writes one half of the combiner's input, whose other half are its queries."""
    g = gen(77)
    for n_src, cols, H, n in ((3, 4, 100, 60), (2, 150, 256, 256), (5, 3, 72, 300)):
        N = n_src * cols
        m = api.memory4(n_src, 40, H).pack(torch.tanh(randn(g, 40, n_src, H, dtype=dtype)))
        lens = torch.randint(1, 41, (n_src,), generator=g, device="cuda", dtype=torch.int32)
        both = randn(g, N, 2 * H + n, dtype=dtype)
        keep = both.clone()
        m.attend(both[:, H:2 * H], lens, out=both[:, :H])
        assert torch.equal(both[:, :H], m.attend(keep[:, H:2 * H].contiguous(), lens)) and torch.equal(both[:, H:], keep[:, H:])
        W = randn(g, n, 2 * H, dtype=dtype) * 0.1
        # (another stride may mean another kernel: the sums of both stray from the exact one, and may be rounded to either side)
        off = 2 * sum_tol(2 * H) * (both[:, :2 * H].double().abs() @ W.double().abs().t()) + 32 * EPS
        want = api.linear(W, both[:, :2 * H].contiguous(), act="tanh")
        api.linear(W, both[:, :2 * H], act="tanh", out=both[:, 2 * H:])
        assert bool(((both[:, 2 * H:].double() - want.double()).abs() <= off + 2 * ref.HALF_STEP[dtype]).all())
        assert torch.equal(both[:, H:2 * H], keep[:, H:2 * H])
        pair = randn(g, N, 2 * n, dtype=dtype)
        R = pair[:, n:].clone()
        api.linear(W, both[:, :2 * H], residual=pair[:, n:], out=pair[:, :n])
        again = api.linear(W, both[:, :2 * H], residual=R)
        assert torch.equal(pair[:, n:], R) and bool(((pair[:, :n].double() - again.double()).abs() <= off + 2 * ref.HALF_STEP[dtype] * (again.double().abs() + off)).all())


def test_rows_that_overlap_are_refused(api):
    one = torch.zeros(1, 64, device="cuda")
    W = torch.zeros(8, 64, device="cuda")
    lens = torch.ones(2, dtype=torch.int32, device="cuda")
    m = api.memory4(2, 3, 64).pack(torch.zeros(3, 1, 64, device="cuda").expand(3, 2, 64))  # (read only: a column for all is fine)
    for call in (lambda: api.linear(W, one.expand(5, 64)), lambda: api.linear(one.expand(5, 64), W), lambda: api.linear(W, W, out=torch.zeros(1, 8, device="cuda").expand(8, 8)),
                 lambda: api.beam_select(one.expand(4, 64), torch.zeros(4, device="cuda"), 2, 2), lambda: m.attend(one.expand(4, 64), lens),
                 lambda: api.linear(W, W.as_strided((4, 64), (32, 1)))):
        with pytest.raises((api.ZrnnError, ValueError)):
            call()
