"""The operators of a decoding step that a host program runs beside the layer objects, as cases that can be timed: the source memory held
in 4 bits (`memory4`: pack, unpack, attend), the product with bias, activation and residual (`linear`), and the selection over
beams and vocabulary with the reorder of the states (`beam_select`, `beam_reorder`).

Where `own` is false, `run` computes them from elementary torch operations; where it is true, it makes the calls of this library.
Tensors lie as they do in the rest of the library: hidden vectors contiguous, one per column; a sequence of states is [slot][column][H].
"""
import math

import numpy as np  # noqa: F401
import torch

own = False

_TYPE = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}
_SEVENTH = 0.14285714924335479736328125  # 1/7 rounded to 32 bits
_MAX_SCALE = 9352.0  # the largest half-precision number that times 7 is one
_ACTS = ("none", "tanh", "sigmoid", "relu", "gelu", "silu")


# ------------------------------------------------------------------------------------------------ the cases
def _memory(name, B, S, heads, d, dtype):
    """B sentences of S slots each: `heads` vectors of d elements per slot."""
    return dict(name=name, kind="memory", B=B, S=S, heads=heads, d=d, dtype=dtype)


def _attend(name, B, C, s_min, S, heads, d, dtype, empty=0):
    """C target columns for each of B sentences of s_min .. S words in S slots; `empty` sentences have no word at all."""
    return dict(name=name, kind="attend", B=B, C=C, s_min=s_min, S=S, heads=heads, d=d, dtype=dtype, empty=empty)


def _linear(name, n, K, N, act, dtype, bias=True, residual=False, pad=0):
    """n outputs from K inputs for N columns; rows of all matrices are `pad` elements further apart than they are long."""
    return dict(name=name, kind="linear", n=n, K=K, N=N, act=act, dtype=dtype, bias=bias, residual=residual, pad=pad)


def _beam(name, B, beam, V, H, layers, dtype, lse, done=0.0):
    """B sentences of `beam` hypotheses over V words, k = beam survivors; the states of `layers` layers of H units move along."""
    return dict(name=name, kind="beam", B=B, beam=beam, V=V, H=H, layers=layers, dtype=dtype, lse=lse, done=done)


def listed():
    return [
        # the encoder's states of a minibatch of sentences, put into 4 bits once per batch and read back
        _memory("memory_batch", 64, 50, 1, 1000, "f32"),
        # the same for long documents: the largest memory
        _memory("memory_long", 16, 8192, 1, 1024, "bf16"),
        # interactive translation: one sentence, the default beam; the smallest call, where latency counts
        _attend("attend_single", 1, 12, 23, 23, 1, 1000, "f32"),
        # a batch of ragged sentences under the default beam
        _attend("attend_batch", 64, 12, 10, 50, 1, 1000, "f32"),
        # a batch of long documents: the memory is far larger than what a step computes with it
        _attend("attend_long", 16, 12, 4000, 8192, 1, 1024, "bf16"),
        # several heads over a memory of paragraphs, some of them empty
        _attend("attend_heads", 32, 5, 100, 1500, 8, 64, "f16", empty=2),
        # the attention's combiner for a decoding batch: tanh(W [c; h] + b)
        _linear("linear_combiner", 1000, 2000, 768, "tanh", "f32"),
        # one step of one sentence's beam: the weights pass by a handful of columns
        _linear("linear_step", 4000, 1000, 12, "sigmoid", "bf16"),
        # all target positions of a minibatch at once, with a residual connection: the largest product
        _linear("linear_large", 8192, 2048, 16384, "gelu", "bf16", residual=True),
        # selection and state reorder of one sentence
        _beam("beam_single", 1, 12, 40000, 1000, 2, "f32", lse=True),
        # of a batch of sentences, some hypotheses finished
        _beam("beam_batch", 64, 12, 50000, 1000, 4, "f32", lse=True, done=0.2),
        # a large vocabulary in 16 bits, log-probabilities rather than logits
        _beam("beam_large", 128, 8, 200000, 2048, 2, "bf16", lse=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


_LIMIT = {  # (bytes, operations) of the largest listed case of each kind
    "memory": (6.1e8, 1e18), "attend": (5.6e7, 4.7e9), "linear": (6.4e8, 5.4e11), "beam": (4.9e8, 1e18)}


def draw(rng):
    while True:
        c = _draw(rng)
        w = work(c)
        if w["bytes"] <= _LIMIT[c["kind"]][0] and w["flops"] <= _LIMIT[c["kind"]][1]:
            c.pop("name")
            return c


def _draw(rng):
    kind = rng.choice(["memory", "attend", "attend", "linear", "linear", "linear", "beam", "beam"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if kind in ("memory", "attend"):
        heads = rng.choice([1, 1, 2, 4, 8, 16])
        d = _log_int(rng, 20, 1024) if heads == 1 else _log_int(rng, 16, 256)
        if rng.random() < 0.4:
            d = max(32, d // 32 * 32)
        B, S = _log_int(rng, 1, 512), _log_int(rng, 1, 16384)
        if kind == "memory":
            return _memory("", B, S, heads, d, dtype)
        return _attend("", B, rng.choice([1, 1, _log_int(rng, 2, 16), _log_int(rng, 2, 40)]), rng.choice([1, max(1, S // 4), S]), S, heads, d, dtype,
                       empty=rng.choice([0, 0, 1]) if B > 1 else 0)
    if kind == "linear":
        n, K, N = _log_int(rng, 32, 16384), _log_int(rng, 32, 8192), _log_int(rng, 1, 16384)
        if rng.random() < 0.6:
            n, K = max(8, n // 8 * 8), max(8, K // 8 * 8)
        return _linear("", n, K, N, rng.choice(_ACTS), dtype, bias=rng.random() < 0.8, residual=rng.random() < 0.4, pad=rng.choice([0, 0, 0, 8, 24, 3]))
    return _beam("", _log_int(rng, 1, 256), rng.choice([1, 2, 4, 5, 8, 10, 12, 12, 16, 24, 32]), _log_int(rng, 700, 200000), 4 * _log_int(rng, 16, 512),
                 rng.choice([1, 2, 4]), dtype, lse=rng.random() < 0.5, done=rng.choice([0.0, 0.3]))


# ------------------------------------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _lengths(case, gen):
    """Sentence lengths spread over s_min .. S, the longest among them, in an order of the seed's; the first `empty` of them 0."""
    B = case["B"]
    n = torch.linspace(case["S"], case["s_min"], B, device="cuda").round().to(torch.int32)
    n = n[torch.randperm(B, generator=gen, device="cuda")].clone()
    n[:case["empty"]] = 0
    return n


def _states(case, gen):
    """States of an LSTM: within -1 .. 1, most of them small; [S][B][heads * d]."""
    return torch.tanh(0.5 * _normal(gen, case["S"], case["B"], case["heads"] * case["d"])).to(_TYPE[case["dtype"]])


def prepare(case, seed):
    gen, t, kind = _generator(seed), _TYPE[case["dtype"]], case["kind"]
    if kind == "memory":
        return dict(case=case, hs=_states(case, gen))
    if kind == "attend":
        hs = _states(case, gen)
        codes, scales = _pack(hs, case["heads"], case["d"])
        lens = _lengths(case, gen)
        q = torch.tanh(_normal(gen, case["B"] * case["C"], case["heads"] * case["d"])).to(t)
        # sources are padded on the left, so a sentence ends in the last slot
        return dict(case=case, codes=codes, scales=scales, lens=lens, offsets=case["S"] - lens, q=q, scale=1.0 if case["heads"] == 1 else case["d"] ** -0.5)
    if kind == "linear":
        n, K, N, pad = case["n"], case["K"], case["N"], case["pad"]
        W = (_normal(gen, n, K + pad) / math.sqrt(K)).to(t)[:, :K]
        X = _normal(gen, N, K + pad).to(t)[:, :K]
        bias = 0.5 * _normal(gen, n) if case["bias"] else None
        R = _normal(gen, N, n + pad).to(t)[:, :n] if case["residual"] else None
        return dict(case=case, W=W, X=X, bias=bias, R=R)
    B, beam, V, H = case["B"], case["beam"], case["V"], case["H"]
    z = torch.empty(B * beam, V, dtype=t, device="cuda")
    lse = torch.empty(B * beam, device="cuda")
    for r in range(0, B * beam, 256):  # (in parts: 32 bits of all rows at once would be much of the card)
        part = 2.0 * _normal(gen, min(256, B * beam - r), V)
        part[:, 1] += 3.0
        l = torch.logsumexp(part, 1)
        z[r:r + 256] = (part if case["lse"] else part - l[:, None]).to(t)
        lse[r:r + 256] = l
    scores = -20.0 + 3.0 * _normal(gen, B * beam)
    done = (torch.rand(B * beam, generator=gen, device="cuda") < case["done"]).to(torch.int32) if case["done"] else None
    n_arrays = 2 * case["layers"] + 1  # h and c of each layer, and the vector that is fed back
    states = [_normal(gen, B * beam, H) for _ in range(n_arrays)]
    return dict(case=case, z=z, lse=lse if case["lse"] else None, scores=scores, done=done, states=states, moved=[torch.empty_like(s) for s in states])


# ------------------------------------------------------------------------------------------------ plain forms
def _groups(x, heads, d):
    """[S][B][heads * d] -> [B][S][heads][groups][32] in 32 bits, zeros behind d."""
    S, B = x.shape[:2]
    x = x.reshape(S, B, heads, d).permute(1, 0, 2, 3).float()
    x = torch.nn.functional.pad(x, (0, -d % 32))
    return x.reshape(B, S, heads, -1, 32)


def _pack(x, heads, d):
    """(codes [B][S][heads][dp / 2], scales [B][S][heads][dp / 32]) of states [S][B][heads * d]."""
    g = _groups(x, heads, d)
    a = g.abs().amax(-1)
    s = torch.clamp(a * torch.tensor(_SEVENTH, device=a.device), max=_MAX_SCALE).half()
    s = torch.where(a <= 3.4028234663852886e38, s, torch.full_like(s, math.nan))
    ok = (s > 0)[..., None]  # (neither zero nor NaN)
    # the quotient in 64 bits: next to the middle between two codes, 32 could end up on it
    q = (g.double() / torch.where(ok, s[..., None].double(), 1.0)).round().clamp(-7, 7)
    u = (torch.where(ok, q, 0.0) + 8).to(torch.uint8)
    u = u.reshape(*u.shape[:3], -1)
    return u[..., 0::2] | (u[..., 1::2] << 4), s


def _values(codes, scales, d):
    """The numbers that the codes stand for, [B][S][heads][d] in 32 bits."""
    u = torch.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:3], -1, 32).float() - 8.0
    v = (u * scales[..., None].float()).half().float()
    return v.reshape(*codes.shape[:3], -1)[..., :d]


def _plain_attend(s, wide):
    case = s["case"]
    B, C, heads, d = case["B"], case["C"], case["heads"], case["d"]
    v = _values(s["codes"], s["scales"], d).to(wide).permute(0, 2, 1, 3)  # [B][heads][S][d]
    q = s["q"].to(wide).reshape(B, C, heads, d).permute(0, 2, 1, 3)
    z = torch.matmul(q, v.transpose(2, 3)) * s["scale"]
    slot = torch.arange(case["S"], device=z.device)
    inside = (slot >= s["offsets"][:, None]) & (slot < (s["offsets"] + s["lens"])[:, None])
    z = torch.where(inside[:, None, None, :], z, -math.inf)
    m = z.amax(-1, keepdim=True)
    p = torch.exp(z - torch.where(m == -math.inf, 0.0, m))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / torch.where(total == 0, 1.0, total)
    return out.permute(0, 2, 1, 3).reshape(B * C, heads * d)


def _plain_act(x, act):
    if act == "tanh":
        return torch.tanh(x)
    if act == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-x))
    if act == "relu":
        return torch.where(x > 0, x, torch.zeros_like(x))
    if act == "gelu":
        return 0.5 * x * (1.0 + torch.erf(x * math.sqrt(0.5)))
    if act == "silu":
        return x / (1.0 + torch.exp(-x))
    return x


def _plain_select(s):
    """(scores, words, parents), each [B][k], best first."""
    case = s["case"]
    B, beam, V = case["B"], case["beam"], case["V"]
    z = s["z"].float()
    if s["lse"] is not None:
        z = z - s["lse"][:, None]
    cand = s["scores"][:, None] + z
    if s["done"] is not None:  # a finished hypothesis proposes itself, once, as word 1
        word = torch.arange(V, device=z.device)
        cand = torch.where(s["done"][:, None] != 0, torch.where(word == 1, s["scores"][:, None], -math.inf), cand)
    cand = torch.where(torch.isnan(cand), -math.inf, cand).view(B, beam * V) + 0.0
    # the order of the values and, among equal ones, of the candidates, in one whole number each
    bits = cand.view(torch.int32).long()
    key = torch.where(bits >= 0, bits, bits ^ 0x7fffffff)
    key = key * 2**32 + (2**32 - 1 - torch.arange(beam * V, device=z.device))
    at = 2**32 - 1 - (torch.topk(key, beam, dim=1).values & (2**32 - 1))
    best = cand.gather(1, at)
    some = best > -math.inf
    word = torch.where(some, at % V, -1).to(torch.int32)
    parent = torch.where(some, at // V + torch.arange(B, device=z.device)[:, None] * beam, -1).to(torch.int32)
    return best, word, parent


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    return _run_own(state) if own else _run_plain(state)


def _run_plain(s):
    case = s["case"]
    t, kind = _TYPE[case["dtype"]], case["kind"]
    if kind == "memory":
        codes, scales = _pack(s["hs"], case["heads"], case["d"])
        return _values(codes, scales, case["d"]).to(t)
    if kind == "attend":
        return _plain_attend(s, torch.float32).to(t)
    if kind == "linear":
        y = torch.matmul(s["X"].float(), s["W"].float().t())
        if s["bias"] is not None:
            y = y + s["bias"]
        y = _plain_act(y, case["act"])
        if s["R"] is not None:
            y = y + s["R"].float()
        return y.to(t)
    best, word, parent = _plain_select(s)
    at = parent.reshape(-1).long()
    moved = [torch.where((at >= 0)[:, None], x[at.clamp(min=0)], 0.0) for x in s["states"]]
    return dict(scores=best, words=word, parents=parent, states=moved)


def _run_own(s):
    from zoph_rnn_b200 import api
    case = s["case"]
    kind = case["kind"]
    if kind == "memory":
        m = api.memory4(case["B"], case["S"], case["d"], heads=case["heads"])
        m.pack(s["hs"])
        return m.unpack(s["hs"].dtype)
    if kind == "attend":
        m = api.memory4(case["B"], case["S"], case["d"], heads=case["heads"], codes=s["codes"], scales=s["scales"])
        return m.attend(s["q"], s["lens"], s["offsets"], scale=s["scale"])
    if kind == "linear":
        return api.linear(s["W"], s["X"], bias=s["bias"], act=case["act"], residual=s["R"])
    best, word, parent = api.beam_select(s["z"], s["scores"], case["beam"], case["beam"], lse=s["lse"], done=s["done"], eos=1)
    moved = api.beam_reorder(s["states"], parent, out=s["moved"])
    return dict(scores=best, words=word, parents=parent, states=moved)


# ------------------------------------------------------------------------------------------------ what a pass needs
def work(case):
    e, kind = _BYTES[case["dtype"]], case["kind"]
    if kind in ("memory", "attend"):
        per = case["heads"] * case["d"]
        packed = case["heads"] * (-(-case["d"] // 32)) * 18  # bytes of a slot: 32 codes and a scale per group
        if kind == "memory":
            return {"bytes": float(case["B"] * case["S"] * (2 * per * e + packed)), "flops": 3.0 * case["B"] * case["S"] * per}
        slots = (case["B"] - case["empty"]) * (case["s_min"] + case["S"]) / 2
        return {"bytes": slots * packed + 2.0 * case["B"] * case["C"] * per * e, "flops": 4.0 * slots * case["C"] * per}
    if kind == "linear":
        n, K, N = case["n"], case["K"], case["N"]
        return {"bytes": float(e * (n * K + K * N + n * N * (2 if case["residual"] else 1)) + (4 * n if case["bias"] else 0)), "flops": 2.0 * n * K * N}
    rows = case["B"] * case["beam"]
    return {"bytes": float(rows * case["V"] * e + rows * case["H"] * (2 * case["layers"] + 1) * 8 + 24 * rows), "flops": 2.0 * rows * case["V"]}


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "memory":
        B, S, heads, d = case["B"], case["S"], case["heads"], case["d"]
        out = torch.empty(B, S, heads, d, dtype=torch.float64, device="cuda")
        x = s["hs"].view(S, B, heads, d)
        for i in range(0, d, 32):  # by the definition, a group at a time
            g = x[..., i:i + 32].double()
            step = (g.abs().amax(-1, keepdim=True).float() * torch.tensor(_SEVENTH, device="cuda")).clamp(max=_MAX_SCALE).half().double()
            code = torch.clamp(torch.round(g / torch.where(step == 0, 1.0, step)), -7.0, 7.0)
            out[..., i:i + 32] = (code * step).half().double().permute(1, 0, 2, 3)
        return out
    if kind == "attend":
        B, C, heads, d, S = case["B"], case["C"], case["heads"], case["d"], case["S"]
        out = torch.zeros(B, C, heads, d, dtype=torch.float64, device="cuda")
        q = s["q"].double().view(B, C, heads, d)
        n = s["lens"].tolist()
        for b in range(B):
            if n[b] == 0:
                continue
            at = slice(S - n[b], S)
            lo, hi = (s["codes"][b, at] & 15).double() - 8, (s["codes"][b, at] >> 4).double() - 8
            v = torch.empty(n[b], heads, 2 * lo.shape[-1], dtype=torch.float64, device="cuda")
            v[..., 0::2], v[..., 1::2] = lo, hi
            v = (v * s["scales"][b, at].double().repeat_interleave(32, -1)).half().double()[..., :d]
            z = torch.einsum("chd,shd->chs", q[b], v) * s["scale"]
            out[b] = torch.einsum("chs,shd->chd", torch.softmax(z, -1), v)
        return out.view(B * C, heads * d)
    if kind == "linear":
        y = torch.einsum("mk,nk->mn", s["X"].double(), s["W"].double())
        if s["bias"] is not None:
            y += s["bias"].double()
        a = case["act"]
        if a == "tanh":
            y = 1 - 2 / (torch.exp(2 * y) + 1)
        elif a == "sigmoid":
            y = torch.exp(-torch.logaddexp(torch.zeros_like(y), -y))
        elif a == "relu":
            y = y.clamp(min=0)
        elif a == "gelu":
            y = y * torch.special.ndtr(y)
        elif a == "silu":
            y = y * torch.exp(-torch.logaddexp(torch.zeros_like(y), -y))
        return y if s["R"] is None else y + s["R"].double()
    B, beam, V = case["B"], case["beam"], case["V"]
    best = []
    for b in range(B):
        at = slice(b * beam, (b + 1) * beam)
        c = s["z"][at].double()
        if s["lse"] is not None:
            c = c - s["lse"][at].double()[:, None]
        c = c + s["scores"][at].double()[:, None]
        if s["done"] is not None:
            over = s["done"][at] != 0
            c[over] = -math.inf
            c[over, 1] = s["scores"][at][over].double()
        best.append(torch.sort(c.reshape(-1), descending=True).values[:beam])
    return dict(scores=torch.stack(best), words=None, parents=None, states=None)
