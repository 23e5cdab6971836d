"""What the operators of a decoding step refuse, before any device is looked for, and the sizes that they name."""
import ctypes

import pytest

from zoph_rnn_b200 import _lib

P = ctypes.c_void_p(1 << 20)  # never followed: the calls below are refused


def at(k):
    return ctypes.c_void_p((1 << 20) + k)


FAR = [ctypes.c_void_p((1 << 40) + (i << 36)) for i in range(12)]


def refused(status, *words):
    L = _lib.lib()
    text = L.zrnn_last_error().decode()
    assert status == _lib.E_ARG, (status, text)
    for w in words:
        assert w in text, text


def size_of(fn, *args):
    n = ctypes.c_size_t()
    assert fn(*args, ctypes.byref(n)) == _lib.OK, _lib.lib().zrnn_last_error()
    return n.value


# ------------------------------------------------------------------ memory4
def test_memory4_sizes():
    L = _lib.lib()
    c, s = ctypes.c_size_t(), ctypes.c_size_t()
    for B, S, h, d in ((1, 1, 1, 1), (3, 7, 1, 33), (64, 50, 1, 1000), (2, 9, 8, 64), (1, 1 << 23, 1, 1024)):
        assert L.zrnn_memory4_sizes(B, S, h, d, ctypes.byref(c), ctypes.byref(s)) == 0
        assert s.value == B * S * h * -(-d // 32) and c.value == 16 * s.value


@pytest.mark.parametrize("bad", [(0, 1, 1, 1), (1, 0, 1, 1), (1, 1, 0, 1), (1, 1, 1, 0), (1, 1, 1 << 16, 1), (1, 1, 1000, 1 << 20), (1 << 22, 1 << 22, 1, 32)])
def test_memory4_sizes_refuses(bad):
    c, s = ctypes.c_size_t(), ctypes.c_size_t()
    refused(_lib.lib().zrnn_memory4_sizes(*bad, ctypes.byref(c), ctypes.byref(s)))
    refused(_lib.lib().zrnn_memory4_sizes(1, 1, 1, 1, None, ctypes.byref(s)), "null")


def test_memory4_of_more_than_2_to_the_30_slots_is_refused():
    """(A window's end, rounded up to whole tiles, has to be an int.)"""
    L = _lib.lib()
    c, s = ctypes.c_size_t(), ctypes.c_size_t()
    assert L.zrnn_memory4_sizes(1, 1 << 30, 1, 32, ctypes.byref(c), ctypes.byref(s)) == _lib.OK
    for S in ((1 << 30) + 1, 2**31 - 1):
        refused(L.zrnn_memory4_sizes(1, S, 1, 32, ctypes.byref(c), ctypes.byref(s)), "slots")
        refused(L.zrnn_memory4_attend_workspace(1, 1, S, 1, 32, ctypes.byref(c)), "slots")
        refused(L.zrnn_memory4_pack(0, P, 32, 32, 1, 1, 1, 32, 0, S, P, P, None), "slots")
        refused(L.zrnn_memory4_unpack(0, P, P, 1, S, 1, 32, 0, 1, P, None), "slots")
        refused(L.zrnn_memory4_attend(0, P, P, 1, S, 1, 32, P, None, FAR[0], 32, 1, None, 1.0, FAR[1], 32, None, 0, None), "slots")


@pytest.mark.parametrize("change, words", [
    (dict(elem=3), "element type"), (dict(elem=-1), "element type"), (dict(S=5, slot0=4), "outside"), (dict(slot0=-1), "outside"),
    (dict(S=-1), "outside"), (dict(S=2**31 - 1, slot0=2**31 - 1), "outside"), (dict(x=None), "null"), (dict(codes=None), "null"),
    (dict(scales=None), "null"), (dict(x=at(2)), "misaligned"), (dict(codes=at(8)), "misaligned"), (dict(scales=at(1)), "misaligned"),
    (dict(ld_slot=-8), "stride"), (dict(heads=0), "positive")])
def test_memory4_pack_refuses(change, words):
    a = dict(elem=0, x=P, ld_slot=96, ld_col=32, S=4, B=3, heads=1, d=32, slot0=0, S_cap=8, codes=P, scales=P) | change
    refused(_lib.lib().zrnn_memory4_pack(*a.values(), None), words)


@pytest.mark.parametrize("change, words", [
    (dict(elem=7), "element type"), (dict(slot0=6), "outside"), (dict(out=None), "null"), (dict(codes=None), "null"), (dict(out=at(1)), "misaligned")])
def test_memory4_unpack_refuses(change, words):
    a = dict(elem=1, codes=P, scales=P, B=3, S_cap=8, heads=2, d=40, slot0=0, S=4, out=P) | change
    refused(_lib.lib().zrnn_memory4_unpack(*a.values(), None), words)


@pytest.mark.parametrize("change, words", [
    (dict(elem=3), "element type"), (dict(d=1025), "1024"), (dict(cols=0), "columns"), (dict(cols=2**31 - 1), "columns"), (dict(codes=None), "null"),
    (dict(lens=None), "null"), (dict(q=None), "null"), (dict(out=None), "null"), (dict(ld_q=31), "leading"), (dict(ld_out=31), "leading"),
    (dict(q=at(2)), "misaligned"), (dict(codes=at(4)), "misaligned"), (dict(out=P, q=P), "overlaps"), (dict(out=at(64), q=P), "overlaps")])
def test_memory4_attend_refuses(change, words):
    a = dict(elem=0, codes=P, scales=P, B=3, S_cap=8, heads=1, d=32, lens=P, offsets=None, q=FAR[0], ld_q=32, cols=2, mask=None, scale=1.0, out=FAR[1],
             ld_out=32, work=None, nwork=0) | change
    refused(_lib.lib().zrnn_memory4_attend(*a.values(), None), words)


def test_memory4_attend_refuses_a_small_workspace():
    L = _lib.lib()
    n = size_of(L.zrnn_memory4_attend_workspace, 1, 12, 1 << 20, 1, 512)
    if n:  # (a long memory of one sentence is cut into parts)
        for w, k in ((None, n), (P, n - 1), (at(4), n)):
            refused(L.zrnn_memory4_attend(0, P, P, 1, 1 << 20, 1, 512, P, None, FAR[0], 512, 12, None, 1.0, FAR[1], 512, w, k, None), "workspace", str(n))


# ------------------------------------------------------------------ linear
@pytest.mark.parametrize("change, words", [
    (dict(elem=3), "element type"), (dict(act=6), "activation"), (dict(act=-1), "activation"), (dict(n=0), "positive"), (dict(K=0), "positive"),
    (dict(N=-1), "positive"), (dict(n=(1 << 24) + 1), "2^24"), (dict(ldw=15), "leading"), (dict(ldx=15), "leading"), (dict(ldy=7), "leading"),
    (dict(R=FAR[3], ldr=7), "leading"), (dict(W=None), "null"), (dict(X=None), "null"), (dict(Y=None), "null"), (dict(W=at(1)), "misaligned"),
    (dict(Y=at(2)), "misaligned"), (dict(bias=at(2)), "misaligned"), (dict(R=at(2), ldr=8), "misaligned"), (dict(Y=FAR[0]), "overlaps"),
    (dict(Y=FAR[1]), "overlaps"), (dict(Y=FAR[2], R=FAR[2], ldr=9), "residual"), (dict(R=ctypes.c_void_p(FAR[2].value + 32), ldr=8), "residual"),
    (dict(bias=FAR[2]), "overlaps")])
def test_linear_refuses(change, words):
    a = dict(elem=0, act=0, n=8, N=5, K=16, W=FAR[0], ldw=16, X=FAR[1], ldx=16, bias=None, R=None, ldr=0, Y=FAR[2], ldy=8, work=None, nwork=0) | change
    refused(_lib.lib().zrnn_linear(*a.values(), None), words)


def test_linear_without_columns_is_nothing():
    assert _lib.lib().zrnn_linear(0, 0, 8, 0, 16, None, 16, None, 16, None, None, 0, None, 8, None, 0, None) == _lib.OK


def test_linear_refuses_a_small_workspace():
    L = _lib.lib()
    for elem in (0, 1, 2):  # rows that no 16-byte copy can start at
        n = size_of(L.zrnn_linear_workspace, elem, 512, 512, 333, FAR[0], 333, FAR[1], 333)
        if n:
            for w, k in ((None, n), (P, n - 1), (at(16), n)):
                refused(L.zrnn_linear(elem, 0, 512, 512, 333, FAR[0], 333, FAR[1], 333, None, None, 0, FAR[2], 512, w, k, None), "workspace", str(n))


# ------------------------------------------------------------------ selection and reorder
@pytest.mark.parametrize("change, words", [
    (dict(elem=5), "element type"), (dict(beam=0), "positive"), (dict(V=0), "positive"), (dict(n=-1), "positive"), (dict(k=0), "k must"), (dict(k=65), "k must"),
    (dict(V=2, k=25), "k must"), (dict(V=1 << 28), "too many"), (dict(ld=99), "leading"), (dict(z=None), "null"), (dict(scores=None), "null"),
    (dict(val=None), "null"), (dict(word=None), "null"), (dict(parent=None), "null"), (dict(done=P, eos=100), "<EOF>"), (dict(done=P, eos=-1), "<EOF>"),
    (dict(z=at(2)), "misaligned"), (dict(val=FAR[0]), "overlaps"), (dict(val=FAR[1]), "overlaps"), (dict(word=FAR[2]), "overlaps"),
    (dict(word=FAR[4], parent=FAR[4]), "overlaps"), (dict(val=FAR[4], parent=FAR[4]), "overlaps")])
def test_beam_select_refuses(change, words):
    a = dict(elem=0, z=FAR[0], ld=100, lse=None, scores=FAR[1], done=None, n=3, beam=12, V=100, k=12, eos=1, val=FAR[2], word=FAR[3], parent=FAR[4], work=None,
             nwork=0) | change
    if "V" in change:
        a["ld"] = change["V"]
    refused(_lib.lib().zrnn_beam_select(*a.values(), None), words)


def test_beam_select_refuses_a_small_workspace():
    L = _lib.lib()
    n = size_of(L.zrnn_beam_select_workspace, 0, 1, 12, 40000, 12)
    if n:
        for w, k in ((None, n), (P, n - 1), (at(8), n)):
            refused(L.zrnn_beam_select(0, FAR[0], 40000, None, FAR[1], None, 1, 12, 40000, 12, 1, FAR[2], FAR[3], FAR[4], w, k, None), "workspace", str(n))


# A workspace that is null, too short by a byte or not aligned; each size asks for one, so that the checks are reached.
@pytest.mark.parametrize("elem", [0, 1, 2])
def test_linear_refuses_a_workspace_that_does_not_do(elem):
    L = _lib.lib()
    n = size_of(L.zrnn_linear_workspace, elem, 4096, 2048, 333, FAR[0], 333, FAR[1], 333)
    assert n >= (4096 + 2048) * 333 * (4 if elem == 0 else 2)  # (both operands are moved)
    for w, k in ((None, n), (P, n - 1), (P, 0), (at(16), n), (at(128), n)):
        refused(L.zrnn_linear(elem, 0, 4096, 2048, 333, FAR[0], 333, FAR[1], 333, None, None, 0, FAR[2], 4096, w, k, None), "workspace", str(n))


@pytest.mark.parametrize("elem, n_sent, beam, V", [(0, 1, 25, 190003), (0, 3, 25, 190003), (1, 2, 50, 200000), (2, 1, 3, 3000001)])
def test_beam_select_refuses_a_workspace_that_does_not_do(elem, n_sent, beam, V):
    L = _lib.lib()
    n = size_of(L.zrnn_beam_select_workspace, elem, n_sent, beam, V, 12)
    assert n >= n_sent * 2 * 12 * 8  # (lists of two CTAs at least)
    for w, k in ((None, n), (P, n - 1), (P, 0), (at(8), n)):
        refused(L.zrnn_beam_select(elem, FAR[0], V, None, FAR[1], None, n_sent, beam, V, 12, 1, FAR[2], FAR[3], FAR[4], w, k, None), "workspace", str(n))


@pytest.mark.parametrize("B, cols, S, heads, d", [(1, 12, 1 << 20, 1, 512), (2, 3, 4000, 2, 64), (3, 4, 4000, 1, 264)])
def test_memory4_attend_refuses_a_workspace_that_does_not_do(B, cols, S, heads, d):
    L = _lib.lib()
    n = size_of(L.zrnn_memory4_attend_workspace, B, cols, S, heads, d)
    assert n >= 2 * B * 16 * d * 4  # (two parts of a source column at least)
    for w, k in ((None, n), (P, n - 1), (P, 0), (at(4), n)):
        refused(L.zrnn_memory4_attend(0, P, P, B, S, heads, d, P, None, FAR[0], heads * d, cols, None, 1.0, FAR[1], heads * d, w, k, None), "workspace", str(n))


def test_beam_select_of_more_than_2_to_the_25_hypotheses_is_refused():
    """(The merge keeps a byte per list, and a list has 1024 rows at most, in shared memory.)"""
    L = _lib.lib()
    c = ctypes.c_size_t()
    assert L.zrnn_beam_select_workspace(0, 1, 1 << 25, 1, 1, ctypes.byref(c)) == _lib.OK and c.value == (1 << 15) * 8
    refused(L.zrnn_beam_select_workspace(0, 1, (1 << 25) + 1, 1, 1, ctypes.byref(c)), "hypotheses")
    refused(L.zrnn_beam_select(0, FAR[0], 1, None, FAR[1], None, 1, (1 << 25) + 1, 1, 1, 1, FAR[2], FAR[3], FAR[4], None, 0, None), "hypotheses")
    assert L.zrnn_beam_select_workspace(0, 1 << 28, 1, 1, 1, ctypes.byref(c)) == _lib.OK and c.value == 0


def byte(p, k):
    return ctypes.c_void_p(p.value + k)


# (on a machine without a device the calls that are let through end there)
@pytest.mark.parametrize("shift, ld, fits", [(128, 64, True), (127 * 4, 160, True), (32 * 4, 160, True), (31 * 4, 160, False), (129 * 4, 160, False), (0, 160, False), (160 * 4 * 2, 160, False), (160 * 4 * 2 + 32 * 4, 160, True), (-128 * 4, 160, True)])
def test_columns_of_one_wider_matrix_do_not_overlap(shift, ld, fits):
    """Queries and outputs, or operands and outputs, side by side in one matrix; columns that share an element are refused."""
    L = _lib.lib()
    for call in (lambda q, o: L.zrnn_memory4_attend(0, P, P, 3, 8, 1, 32, P, None, q, ld, 2, None, 1.0, o, ld, None, 0, None),
                 lambda x, y: L.zrnn_linear(0, 0, 32, 6, 32, FAR[3], 32, x, ld, None, None, 0, y, ld, None, 0, None),
                 lambda r, y: L.zrnn_linear(0, 0, 32, 6, 32, FAR[3], 32, FAR[4], 32, None, r, ld, y, ld, None, 0, None) if shift else _lib.E_ARG):
        status = call(FAR[0], byte(FAR[0], shift))
        assert (status != _lib.E_ARG) == fits, (status, L.zrnn_last_error())
    # a single column within another matrix's; other strides are not looked into
    one = L.zrnn_linear(0, 0, 32, 1, 32, FAR[3], 32, FAR[0], 32, None, byte(FAR[0], 0), 64, byte(FAR[0], 32 * 4), 999, None, 0, None)
    assert one != _lib.E_ARG
    refused(L.zrnn_linear(0, 0, 32, 6, 32, FAR[3], 32, FAR[0], 96, None, None, 0, byte(FAR[0], 128), 160, None, 0, None), "overlaps")


def reorder(src, dst, sizes, n_cols=12, n_src=12, group=12, parents=P):
    k = len(src)
    return _lib.lib().zrnn_beam_reorder(k, (ctypes.c_void_p * k)(*[getattr(s, "value", s) for s in src]), (ctypes.c_void_p * k)(*[getattr(s, "value", s) for s in dst]),
                                        (ctypes.c_size_t * k)(*sizes), parents, n_cols, n_src, group, None)


def test_beam_reorder_refuses():
    a, b, c, d = FAR[:4]
    refused(reorder([a] * 41, [b] * 41, [64] * 41), "40")
    refused(reorder([a], [b], [64], n_cols=-1), "negative")
    refused(reorder([a], [b], [64], parents=None), "null")
    refused(reorder([None], [b], [64]), "null")
    refused(reorder([a], [None], [64]), "null")
    refused(reorder([a], [b], [(1 << 36) + 1]), "2^36")
    refused(reorder([a], [a], [64], n_cols=11), "as many")
    for group in (0, 65, 5, -1):
        refused(reorder([a], [a], [64], group=group), "groups")
    refused(reorder([a], [ctypes.c_void_p(a.value + 64)], [64]), "overlap")
    refused(reorder([a, b], [c, c], [64, 64]), "overlap")
    refused(reorder([a, b], [b, a], [64, 64]), "overlap")
    refused(reorder([a, b], [c, a], [64, 64]), "overlap")
    refused(reorder([a], [P], [64]), "parents")
    assert reorder([], [], []) == _lib.OK
    assert reorder([a], [b], [64], n_cols=0) == _lib.OK


def test_the_wrappers_refuse_tensors_that_do_not_fit():
    import torch
    from zoph_rnn_b200 import api
    z = torch.zeros
    for call in (lambda: api.linear(z(4, 8), z(3, 9)), lambda: api.linear(z(4, 8), z(3, 8, dtype=torch.bfloat16)), lambda: api.linear(z(4, 8), z(3, 8), act="exp"),
                 lambda: api.linear(z(4, 8), z(8, 3).t()), lambda: api.linear(z(4, 8).double(), z(3, 8).double()), lambda: api.linear(z(4, 8), z(3, 8), bias=z(5)),
                 lambda: api.linear(z(4, 8), z(3, 8), residual=z(3, 5)), lambda: api.linear(z(4, 8), z(3, 8), out=z(2, 4)),
                 lambda: api.beam_select(z(10, 7), z(10), 3, 2), lambda: api.beam_select(z(9, 7), z(8), 3, 2), lambda: api.beam_select(z(9, 7), z(9).double(), 3, 2),
                 lambda: api.beam_reorder([z(3, 4)], z(3)), lambda: api.beam_reorder([z(3, 4)], z(3, dtype=torch.int32), out=[z(3, 5)]),
                 lambda: api.beam_reorder([z(4, 3).t()], z(3, dtype=torch.int32), out=[z(3, 4)])):
        with pytest.raises(ValueError):
            call()
