"""The delta rule with kept states over packed sequences (shvk_gdn_step, shvk_gdn_prefill) against the rule in float64, and what it
refuses.

Tolerances.  An output in a 16-bit type is off by half a step of its type, eps / 2 of its value.  Everything else is float32
arithmetic: a product with the state sums DK terms, whose partial sums are rounded up to DK times, and a token adds a dozen roundings
to a state entry; errors carried by the state do not grow, because I - beta k k^T with |k| <= 1 and beta <= 1, and a decay below one,
are contractions.  So an output is within (DK + 16 T) 2^-24 of the largest sum of magnitudes that enters one, |q| |S|, and a state
within the same factor of the largest state column.  The prefill form's pieces are held in 22 bits, which adds two steps of 2^-22
(8 x 2^-24) a chunk: its factor is (DK + 24 T) 2^-24.  Its bf16 outputs come from single fp16 pieces: S cut off to eleven bits (less
than 2^-10 of each entry), and M and U rounded to them (2^-11 each), so that o = M U + Q S0 is off by less than 2^-10 of
sum |M| |U| + |q| |S0| more; that sum, over the up to 64 tokens of a chunk, is taken over the last 64 here, and |q| |S0| over all of
them.
"""
import ctypes as C

import numpy as np
import pytest

from shield_sisa_b200 import binding

CODES = {"fp32": 0, "bf16": 1, "fp16": 2}
INVALID = 1                                                     # cudaErrorInvalidValue


@pytest.fixture(scope="module")
def L():
    from shield_sisa_b200 import build
    build.build()
    return binding.load_library(True)


def call(L, form, a, ws=None, stream=None):
    if form == "step":
        return L.shvk_gdn_step(C.byref(a), stream)
    return L.shvk_gdn_prefill(C.byref(a), ws, L.shvk_gdn_prefill_workspace_bytes(C.byref(a)) if ws else 0, stream)


# ---------------------------------------------------------------------------------------------- refusals (no GPU)
def good(**kw):
    p = 0x100000                                                # never dereferenced: every call below ends on the host
    a = dict(n_seq=2, HK=2, HV=4, DK=64, DV=128, dtype=1, l2norm=1, scale=0.125, n_tokens=9, q=p, ldq=128, k=p, ldk=128, v=p,
             ldv=512, g=p, beta=p, ldgb=4, o=p, ldo=512, seq_start=p, states=p, n_slots=4, slot_in=p, slot_out=p)
    a.update(kw)
    return binding.GdnSeqArgs(**a)


BAD = [dict(n_seq=-1), dict(n_tokens=-1), dict(n_tokens=1 << 31), dict(dtype=3), dict(dtype=-1), dict(DK=96), dict(DK=32),
       dict(DK=256), dict(DV=0), dict(DV=48), dict(DV=288), dict(HK=0), dict(HV=0), dict(HV=5), dict(HK=3), dict(HV=8192),
       dict(seq_start=None), dict(q=None), dict(k=None), dict(v=None), dict(g=None), dict(beta=None), dict(o=None),
       dict(q=0x100008), dict(k=0x100002), dict(v=0x100004), dict(o=0x100008), dict(ldq=129), dict(ldk=132), dict(ldv=514),
       dict(ldo=513), dict(ldo=504), dict(ldq=-128), dict(ldgb=-1), dict(states=None), dict(states=0x100004), dict(n_slots=-1)]


@pytest.mark.parametrize("kw", BAD, ids=lambda d: "-".join(f"{k}={v}" for k, v in d.items()))
def test_step_refuses(L, kw):
    assert call(L, "step", good(**kw)) == INVALID


@pytest.mark.parametrize("kw", BAD + [dict(dtype=0, ldq=128)], ids=lambda d: "-".join(f"{k}={v}" for k, v in d.items()))
def test_prefill_refuses(L, kw):
    a = good(**kw)
    assert L.shvk_gdn_prefill(C.byref(a), 0x200000, 1 << 40, None) == INVALID
    if "dtype" not in kw:
        assert L.shvk_gdn_prefill_workspace_bytes(C.byref(a)) == 0


@pytest.mark.parametrize("form", ["step", "prefill"])
@pytest.mark.parametrize("kw", [{name: 0x100000 + off} for name in ("g", "beta", "seq_start", "slot_in", "slot_out") for off in (1, 2, 3)] + [dict(ldgb=1 << 33)], ids=str)
def test_refuses_arrays_that_no_word_is_read_from(L, form, kw):
    """Float32 and int32 arrays that do not start on four bytes: a read would fault."""
    a = good(**kw)
    ws = 0x200000
    assert (L.shvk_gdn_step(C.byref(a), None) if form == "step" else L.shvk_gdn_prefill(C.byref(a), ws, 1 << 40, None)) == INVALID
    assert L.shvk_gdn_prefill_workspace_bytes(C.byref(a)) == 0


def test_starved_launch_refuses_what_waits_for_nothing(L):
    a = good(DV=64, ldv=256, ldo=256)
    assert L.shvk_gdn_prefill_starved(C.byref(a), 0x200000, 1 << 40, 256, None) == INVALID
    assert L.shvk_gdn_prefill_starved(None, 0x200000, 1 << 40, 256, None) == INVALID
    assert L.shvk_gdn_prefill_status(None) == INVALID


def test_prefill_refuses_its_workspace(L):
    a = good()
    need = L.shvk_gdn_prefill_workspace_bytes(C.byref(a))
    assert need >= 4 * 3 * 2048                                 # 4 heads; 9 rows of two sequences take three chunks at most
    for ws, size in ((None, need), (0x200008, need), (0x200000, need - 1), (0x200000, 0)):
        assert L.shvk_gdn_prefill(C.byref(a), ws, size, None) == INVALID
    assert L.shvk_gdn_prefill(C.byref(good(n_seq=0)), None, 0, None) == 0
    assert L.shvk_gdn_prefill_workspace_bytes(C.byref(good(n_seq=0))) == 0
    assert L.shvk_gdn_prefill_workspace_bytes(None) == 0 and L.shvk_gdn_prefill(None, 0x200000, need, None) == INVALID


def test_prefill_needs_no_more_than_a_program_keeps_for_it(L):
    """One piece for calls of any lengths, as the header promises it: 8,192 bytes of a value head for every 16 rows and every sequence."""
    import random
    rng = random.Random(4)
    log = lambda hi: int(hi ** rng.random())  # noqa: E731
    segments = False
    for i in range(20000):
        n, hk, dk, dv, dtype = log(600), rng.choice([1, 2, 6]), rng.choice([64, 128]), rng.choice([32, 64, 96, 128, 128]), rng.choice([1, 2])
        tokens, hv = n * log(20000) + rng.choice([0, 0, 3, 63]), hk * rng.choice([1, 2, 3])
        a = good(n_seq=n, HK=hk, HV=hv, DK=dk, DV=dv, dtype=dtype, n_tokens=tokens, ldq=hk * dk, ldk=hk * dk, ldv=hv * dv, ldo=hv * dv, ldgb=hv)
        need = L.shvk_gdn_prefill_workspace_bytes(C.byref(a))
        assert 0 < need <= hv * (tokens // 16 + n + 1) * 8192, (n, hv, dk, dv, dtype, tokens)
        segments |= need > 22032 * (tokens // 64 + n) * hv and dv > 64
    assert segments                                             # calls that keep states of segments were among them


def test_prefill_needs_nothing_for_a_type_that_it_refuses(L):
    a = good(dtype=0)
    assert L.shvk_gdn_prefill_workspace_bytes(C.byref(a)) == 0 and L.shvk_gdn_prefill(C.byref(a), 0x200000, 1 << 40, None) == INVALID


def test_step_of_nothing_launches_nothing(L):
    assert L.shvk_gdn_step(None, None) == INVALID
    assert call(L, "step", good(n_seq=0)) == 0
    assert call(L, "step", good(n_seq=0, seq_start=None, q=None)) == 0


# ---------------------------------------------------------------------------------------------- GPU
gpu = pytest.mark.gpu
LAYOUTS = [(6, 6, 64, 128), (2, 6, 128, 128), (1, 4, 64, 64), (2, 2, 128, 256), (3, 3, 64, 32), (1, 1, 128, 96)]


def make(kind, lens, hk, hv, dk, dv, seed, tail=3, fused=False, unit=False, slots=None):
    """A call's buffers: packed rows (separate, or slices of one fused row), states, slots."""
    import torch
    t = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}[kind]
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    n, rows = len(lens), sum(lens) + tail
    x = {"n": n, "lens": lens, "hk": hk, "hv": hv, "dk": dk, "dv": dv, "kind": kind, "rows": rows, "l2norm": not unit, "scale": dk ** -0.5}
    widths = [hk * dk, hk * dk, hv * dv]
    if fused:                                                   # q | k | v | something else
        row = rn(rows, sum(widths) + 40).to(t)
        parts = list(row.split(widths + [40], 1)[:3])
    else:
        parts = [rn(rows, w).to(t) for w in widths]
    if unit:
        for i in range(2):
            p = parts[i].float().reshape(rows, hk, dk)
            parts[i] = (p / p.norm(dim=-1, keepdim=True).clamp_min(1e-3)).reshape(rows, -1).to(t)
    x["q"], x["k"], x["v"] = parts
    x["g"] = -torch.exp(rn(rows, hv) - 2.0)
    x["beta"] = torch.sigmoid(rn(rows, hv))
    x["o"] = torch.full((rows, hv, dv), 7.0, device="cuda").to(t)
    starts = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    x["seq_start"] = torch.from_numpy(starts).cuda()
    x["n_slots"] = 2 * n + 1
    x["states"] = rn(x["n_slots"], hv, dk, dv)
    x["slot_in"] = torch.arange(n, device="cuda", dtype=torch.int32) if slots is None else slots[0]
    x["slot_out"] = (n + torch.randperm(n, device="cuda", generator=gen)).to(torch.int32) if slots is None else slots[1]
    return x


def args(x):
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    return binding.GdnSeqArgs(n_seq=x["n"], HK=x["hk"], HV=x["hv"], DK=x["dk"], DV=x["dv"], dtype=CODES[x["kind"]],
                              l2norm=int(x["l2norm"]), scale=x["scale"], n_tokens=x["rows"], q=ptr(x["q"]), ldq=x["q"].stride(0),
                              k=ptr(x["k"]), ldk=x["k"].stride(0), v=ptr(x["v"]), ldv=x["v"].stride(0), g=ptr(x["g"]),
                              beta=ptr(x["beta"]), ldgb=x["g"].stride(0), o=ptr(x["o"]), ldo=x["o"].stride(0),
                              seq_start=ptr(x["seq_start"]), states=ptr(x["states"]), n_slots=x["n_slots"], slot_in=ptr(x["slot_in"]),
                              slot_out=ptr(x["slot_out"]))


def launch(L, form, x, stream=None):
    """The call on the current (or the given) stream; the prefill form's workspace is poisoned: it must not rely on its contents."""
    import torch
    s = torch.cuda.current_stream() if stream is None else stream
    a, ws = args(x), None
    if form == "prefill":
        need = L.shvk_gdn_prefill_workspace_bytes(C.byref(a))
        if "ws" not in x or x["ws"].numel() < need:
            x["ws"] = torch.full((max(need, 16),), 0xff, device="cuda", dtype=torch.uint8)
        ws = x["ws"].data_ptr()
    rc = call(L, form, a, ws, s.cuda_stream)
    assert rc == 0, rc


def rule(x, state0):
    """o [rows, hv, dv] (7 where no sequence has a row), the state behind each sequence, |q| |S| at most, in float64; x["pieces"]: the most
    that |M| |U| + |q| |S0| of a chunk can be."""
    import torch
    hk, hv, dk, dv, group = x["hk"], x["hv"], x["dk"], x["dv"], x["hv"] // x["hk"]
    q = x["q"].double().reshape(x["rows"], hk, dk)
    k = x["k"].double().reshape(x["rows"], hk, dk)
    v = x["v"].double().reshape(x["rows"], hv, dv)
    if x["l2norm"]:
        q, k = (z / torch.sqrt((z * z).sum(-1, keepdim=True) + 1e-6) for z in (q, k))
    q = q * float(np.float32(x["scale"]))
    q, k = q.repeat_interleave(group, 1), k.repeat_interleave(group, 1)
    o = torch.full((x["rows"], hv, dv), 7.0, device="cuda", dtype=torch.float64)
    out, big, x["pieces"] = [], 0.0, 0.0
    row = 0
    for n, ln in enumerate(x["lens"]):
        S = state0[n].double().clone()
        last, size = [], [S.norm(dim=1)]
        for _ in range(ln):
            S = S * torch.exp(x["g"][row].double())[:, None, None]
            u = x["beta"][row].double()[:, None] * (v[row] - torch.einsum("hk,hkv->hv", k[row], S))
            S = S + k[row][:, :, None] * u[:, None, :]
            o[row] = torch.einsum("hk,hkv->hv", q[row], S)
            big = max(big, float((q[row].norm(dim=-1)[:, None] * S.norm(dim=1)).max()))
            last, size = last[-63:] + [(k[row], u.abs())], size[-64:] + [S.norm(dim=1)]
            ks, us = torch.stack([z[0] for z in last]), torch.stack([z[1] for z in last])
            mixed = torch.einsum("hj,jhv->hv", torch.einsum("hk,jhk->hj", q[row], ks).abs(), us)
            x["pieces"] = max(x["pieces"], float((mixed + q[row].norm(dim=-1)[:, None] * torch.stack(size).amax(0)).max()))
            row += 1
        out.append(S)
    return o, out, big


def first_states(x):
    import torch
    ids = [-1] * x["n"] if x["slot_in"] is None else x["slot_in"].tolist()
    return [x["states"][i].clone() if 0 <= i < x["n_slots"] else torch.zeros_like(x["states"][0]) for i in ids]


def check(L, form, x, **kw):
    """Runs the call and compares all of its outputs, the rows and slots that it must leave alone among them."""
    import torch
    first, pool = first_states(x), x["states"].clone()
    want, states, big = rule(x, first)
    launch(L, form, x, **kw)
    torch.cuda.synchronize()
    total, longest = sum(x["lens"]), max(x["lens"] + [0])
    factor = (x["dk"] + (16 if form == "step" else 24) * longest) * 2.0 ** -24
    half = torch.finfo(x["o"].dtype).eps / 2
    got = x["o"].double()
    tiny = 2.0 ** -25 if x["kind"] == "fp16" else 0.0            # half a step of fp16's subnormal numbers
    most = torch.finfo(x["o"].dtype).max
    single = 2.0 ** -10 * x["pieces"] if form == "prefill" and x["kind"] == "bf16" else 0.0
    tol = factor * big + single + tiny + half * want.abs()
    over, near = want.abs() - tol > 1.01 * most, want.abs() + tol > 0.99 * most
    assert torch.equal(got[over], torch.inf * want[over].sign())  # what the type cannot hold is infinite in it
    off = torch.where(near, 0, (got - want).abs() - tol)         # (and may be where it nearly cannot)
    assert float(off[:total].max()) <= 0 if total else True
    assert torch.equal(x["o"][total:], torch.full_like(x["o"][total:], 7.0))
    written = {}
    for n, s in enumerate([] if x["slot_out"] is None else x["slot_out"].tolist()):
        if 0 <= s < x["n_slots"]:
            written[s] = n
    for s in range(x["n_slots"]):
        if s not in written:
            assert torch.equal(x["states"][s], pool[s])
            continue
        n = written[s]
        if x["lens"][n] == 0:
            assert torch.equal(x["states"][s], first[n])
            continue
        column = max(float(states[n].norm(dim=1).max()), float(first[n].double().norm(dim=1).max()))
        assert float((x["states"][s].double() - states[n]).abs().max()) <= factor * column
    return got, states


@gpu
@pytest.mark.parametrize("kind", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("layout", LAYOUTS, ids=str)
@pytest.mark.parametrize("lens", [[1], [1] * 7, [3, 0, 1, 8], [0], [33]], ids=str)
def test_step(L, kind, layout, lens):
    check(L, "step", make(kind, lens, *layout, seed=len(lens) + layout[2]))


@gpu
@pytest.mark.parametrize("kind", ["fp32", "bf16"])
def test_step_on_slices_of_one_row_without_normalising(L, kind):
    check(L, "step", make(kind, [2, 5, 1], 2, 4, 64, 128, seed=5, fused=True, unit=True))


LENGTHS = [[1], [16], [17, 15], [0, 1, 33, 48], [0], [79], [130, 2, 64, 0, 0, 31]]


@gpu
@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("layout", LAYOUTS, ids=str)
@pytest.mark.parametrize("lens", LENGTHS, ids=str)
def test_prefill(L, kind, layout, lens):
    check(L, "prefill", make(kind, lens, *layout, seed=len(lens) + layout[2]))


@gpu
@pytest.mark.parametrize("kind", ["bf16", "fp16"])
def test_prefill_on_slices_of_one_row_without_normalising(L, kind):
    check(L, "prefill", make(kind, [70, 5, 1], 2, 4, 64, 128, seed=5, fused=True, unit=True))
    check(L, "prefill", make(kind, [70, 5, 1], 2, 4, 128, 128, seed=6, fused=True))


@gpu
@pytest.mark.parametrize("n", [1, 30, 60, 200])
def test_prefill_of_few_and_many_sequences(L, n):
    """Short sequences: every share of the value columns that a CTA of the 16-token form may take: the same bits in all."""
    import torch
    x = make("bf16", [50] * n, 2, 4, 128, 128, seed=8, tail=0)
    for name in ("q", "k", "v", "g", "beta"):
        x[name][:50 * n] = x[name][:50].repeat(n, 1)
    x["states"][:n] = x["states"][0].clone()
    y = make("bf16", [50], 2, 4, 128, 128, seed=8, tail=0)
    for name in ("q", "k", "v", "g", "beta"):
        y[name][:50] = x[name][:50]
    y["states"][0] = x["states"][0]
    check(L, "prefill", y)
    launch(L, "prefill", x)
    torch.cuda.synchronize()
    for i in range(n):
        assert torch.equal(x["o"][50 * i:50 * i + 50], y["o"][:50])
    assert torch.equal(x["states"][x["slot_out"].long()], y["states"][1:2].expand(n, -1, -1, -1))


@gpu
@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("what", ["tiny_values", "huge_values", "huge_state", "tiny_state", "rising", "falling", "vanishing", "large_keys", "small_keys", "no_decay"])
def test_prefill_of_any_size_of_numbers(L, kind, what):
    """The scales of the pieces follow the numbers: a state or values far from one, that grow or fade by many powers of two on the way,
    keys and queries that are normalised from far away."""
    import torch
    x = make(kind, [300, 45], 2, 4, 64, 128, seed=17)
    far = 1e-4 if kind == "fp16" else 1e-12
    at = torch.arange(x["rows"], device="cuda", dtype=torch.float32)[:, None]
    t = x["v"].dtype
    if what == "tiny_values":
        x["v"] = (x["v"].float() * far).to(t)
        x["states"] *= far
    elif what == "huge_values":
        x["v"] = (x["v"].float() * (1e3 if kind == "fp16" else 1e12)).to(t)
    elif what == "huge_state":
        x["states"] *= 1e15
    elif what == "tiny_state":
        x["states"] *= 1e-15
    elif what == "rising":
        x["v"] = (x["v"].float() * torch.exp(-4 + at / 25)).to(t)
    elif what == "falling":
        x["v"] = (x["v"].float() * torch.exp(4 - at / 25)).to(t)
        x["g"] -= 0.2
    elif what == "vanishing":                                   # no values any more, and a state that fades to nothing
        x["v"][100:] = 0
        x["g"] -= 0.8
    elif what == "large_keys":
        x["k"], x["q"] = (x["k"].float() * 1000).to(t), (x["q"].float() * 300).to(t)
    elif what == "small_keys":
        x["k"], x["q"] = (x["k"].float() * 0.01).to(t), (x["q"].float() * 0.02).to(t)
    else:
        x["g"] *= 0
    check(L, "prefill", x)


@gpu
@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("layout,lens", [((1, 1, 128, 128), [4099]), ((1, 2, 64, 128), [3000, 64 * 13 * 3]), ((1, 1, 128, 256), [2496]),
                                         ((1, 1, 128, 64), [4000]), ((1, 1, 64, 192), [70, 5100]),
                                         ((1, 1, 64, 128), [0, 5000, 1, 900]), ((1, 1, 64, 128), [0, 9000, 1, 2000])], ids=str)
def test_few_long_sequences_are_walked_in_segments(L, kind, layout, lens):
    """Segments of at least 13 chunks: whole ones, a last one of a few tokens, sequences of one segment and of none among them; states
    left where they were read from."""
    import torch
    x = make(kind, lens, *layout, seed=61)
    x["g"] *= 0.1
    x["slot_out"] = x["slot_in"].clone()
    chunks = (16912 if kind == "bf16" else 22032) * (x["rows"] // 64 + x["n"] + 1) * layout[1]
    segments = L.shvk_gdn_prefill_workspace_bytes(C.byref(args(x))) - chunks > 4 * layout[2] * layout[3]      # room for their states
    assert segments == (sum(lens) / len(lens) >= 39 * 64)         # by the average: three of 13 chunks at least (two are walked one after the other)
    check(L, "prefill", x)


@gpu
def test_segments_of_a_sequence_that_begins_behind_the_first_row(L):
    import torch
    x = make("bf16", [200, 3300], 1, 1, 128, 128, seed=63)
    y = make("bf16", [200, 3300], 1, 1, 128, 128, seed=63)
    y["n"], y["lens"] = 1, [3300]
    for name in ("seq_start", "slot_in", "slot_out"):
        y[name] = y[name][1:].clone()
    first = x["states"][1:2].clone()
    z = {**x, "q": x["q"][200:], "k": x["k"][200:], "v": x["v"][200:], "g": x["g"][200:], "beta": x["beta"][200:], "lens": [3300], "rows": 3303}
    want, states, big = rule(z, first)
    launch(L, "prefill", y)
    torch.cuda.synchronize()
    factor = (128 + 24 * 3300) * 2.0 ** -24
    got = y["o"][200:].double()
    assert float(((got - want).abs() - 2.0 ** -8 * want.abs())[:3300].max()) <= factor * big + 2.0 ** -10 * z["pieces"]
    assert torch.equal(y["o"][:200], torch.full_like(y["o"][:200], 7.0))
    s = y["states"][int(y["slot_out"][0])].double()
    assert float((s - states[0]).abs().max()) <= factor * float(states[0].norm(dim=1).max())


@gpu
def test_not_a_number_in_a_segment_stays_in_its_column_and_behind(L):
    import torch
    x, y = (make("bf16", [3900], 1, 1, 128, 128, seed=65) for _ in range(2))
    x["v"][2000, 5] = float("nan")
    launch(L, "prefill", x)
    launch(L, "prefill", y)
    torch.cuda.synchronize()
    assert torch.isnan(x["o"][2000:3900, 0, 5].float()).all() and torch.isfinite(x["o"][:2000].float()).all()
    keep = torch.arange(128, device="cuda") != 5
    assert torch.equal(x["o"][:, 0, keep], y["o"][:, 0, keep])
    assert torch.equal(x["states"][1][0][:, keep], y["states"][1][0][:, keep]) and torch.isnan(x["states"][1][0][:, 5]).all()


@gpu
def test_step_continues_what_prefill_left(L):
    """A prompt by the chunked form, then token after token in place, against one walk over all of it; and the two forms agree."""
    import torch
    lens, new = [65, 1, 40], 5
    whole = make("bf16", [n + new for n in lens], 2, 4, 128, 128, seed=23, tail=0)
    want, states, big = rule(whole, first_states(whole))
    starts = np.concatenate([[0], np.cumsum([n + new for n in lens])])
    factor = (128 + 24 * 70) * 2.0 ** -24

    def part(pick, n_rows):
        x = dict(whole)
        idx = torch.tensor(pick, device="cuda")
        for name in ("q", "k", "v", "g", "beta"):
            x[name] = whole[name][idx].contiguous()
        x["rows"], x["lens"] = len(pick), n_rows
        x["o"] = torch.full((len(pick), 4, 128), 7.0, device="cuda").to(whole["o"].dtype)
        x["seq_start"] = torch.from_numpy(np.concatenate([[0], np.cumsum(n_rows)]).astype(np.int32)).cuda()
        return x
    pick = [starts[i] + j for i, n in enumerate(lens) for j in range(n)]
    x = part(pick, lens)
    x.pop("ws", None)
    launch(L, "prefill", x)
    half = 2.0 ** -8
    ref = want[torch.tensor(pick, device="cuda")]
    assert float(((x["o"].double() - ref).abs() - half * ref.abs()).max()) <= factor * big + 2.0 ** -10 * whole["pieces"]
    for j in range(new):
        pick = [starts[i] + n + j for i, n in enumerate(lens)]
        y = part(pick, [1] * 3)
        y["slot_in"] = whole["slot_out"]
        launch(L, "step", y)
        ref = want[torch.tensor(pick, device="cuda")]
        assert float(((y["o"].double() - ref).abs() - half * ref.abs()).max()) <= factor * big
    for i in range(3):
        got = whole["states"][int(whole["slot_out"][i])].double()
        assert float((got - states[i]).abs().max()) <= factor * float(states[i].norm(dim=1).max())


@gpu
@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("dk", [64, 128])
def test_prefill_keeps_float32_over_a_long_sequence(L, kind, dk):
    """4,099 tokens with next to no decay: 257 chunks' sums.  As norms, where roundings do not add up but their squares do, the state is
    within 1e-6 of float64 and an output within 1.3 half steps' rms of its type (eps / 2 / sqrt 3 over a mantissa of 1.4 on average)."""
    import torch
    x = make(kind, [4099], 1, 1, dk, 128, seed=29)
    x["g"] *= 0.01
    want, states, _ = rule(x, first_states(x))
    launch(L, "prefill", x)
    torch.cuda.synchronize()
    s = x["states"][int(x["slot_out"][0])].double()
    rel_s = float((s - states[0]).norm() / states[0].norm())
    rel_o = float((x["o"][:4099].double() - want[:4099]).norm() / want[:4099].norm())
    rms = torch.finfo(x["o"].dtype).eps / 2 / 3 ** 0.5 / 1.4
    print(f"state {rel_s:.2e}, outputs {rel_o:.2e} (rounding alone {rms:.2e})")
    assert rel_s < 1e-6 and rel_o < 1.3 * rms


def slot_cases():
    return {"none": (None, None), "in_place": ([2, 0, 4], [2, 0, 4]), "new": ([-1, -1, -1], [1, 5, 3]), "not_kept": ([3, 1, 1], [-1, -1, -1]),
            "mixed": ([0, -1, 0], [1, 2, -1]), "outside": ([7, 1 << 30, -5], [3, 7, 1 << 30])}


@gpu
@pytest.mark.parametrize("form", ["step", "prefill"])
@pytest.mark.parametrize("name", list(slot_cases()))
def test_slots(L, form, name):
    """States read from and left in the slots that are named, by whom; a slot read by many; values that are no slot."""
    import torch
    s = tuple(None if v is None else torch.tensor(v, device="cuda", dtype=torch.int32) for v in slot_cases()[name])
    for lens in ([1, 1, 1], [0, 3, 20]):
        check(L, form, make("bf16", lens, 2, 4, 64, 128, seed=3, slots=s))
    if name == "none":
        x = make("bf16", [2, 3, 1], 2, 4, 64, 128, seed=3, slots=s)
        x["states"], keep = None, x["states"]
        a = binding.GdnSeqArgs.from_buffer_copy(args({**x, "states": keep}))
        a.states, a.n_slots = None, 0
        assert call(L, form, a, None if form == "step" else x.setdefault("ws", torch.empty(1 << 22, device="cuda", dtype=torch.uint8)).data_ptr(),
                    torch.cuda.current_stream().cuda_stream) == 0
        want = rule(x, [torch.zeros_like(keep[0])] * 3)
        assert float((x["o"].double() - want[0]).abs().max()) < 0.02 * float(want[0][:6].abs().max())


@gpu
@pytest.mark.parametrize("form", ["step", "prefill"])
def test_bounds_of_sequences_that_are_no_bounds(L, form):
    """Starts outside the rows are cut to them: nothing outside the caller's rows is touched, and the sequences that are well described
    are right."""
    import torch
    x = make("bf16", [4, 3, 5], 2, 4, 64, 128, seed=9, tail=0)
    x["seq_start"] = torch.tensor([0, 4, -9, 1 << 30], device="cuda", dtype=torch.int32)      # 4 rows; none; all 12
    guard = x["states"][2 * x["n"]].clone()
    launch(L, form, x)
    torch.cuda.synchronize()
    y = make("bf16", [4, 3, 5], 2, 4, 64, 128, seed=9, tail=0)
    y["lens"], y["n"] = [4], 1
    assert torch.equal(x["states"][2 * x["n"]], guard)
    y["seq_start"] = x["seq_start"][:2].clone()
    before = y["states"].clone()
    launch(L, form, y)
    torch.cuda.synchronize()
    slot = int(x["slot_out"][0])
    assert torch.equal(x["states"][slot], y["states"][slot]) and not torch.equal(y["states"][slot], before[slot])


@gpu
@pytest.mark.parametrize("form", ["step", "prefill"])
def test_a_decay_to_nothing_forgets_everything(L, form):
    """g = -inf and g = the type's lowest value: what follows does not depend on the state before, not even where that is huge.  The
    prefill form holds a chunk's 64 values of W = V - e K S0 in a column to 2^-32 of the largest: with a state of `fill`, W before the
    reset is at most 8 fill (|k|_1 <= sqrt 64), so U behind it is off by up to 64 x 8 x 2^-32 fill, and what 64 of those make of an
    output or a state (each times at most 1) by 2^-17 fill."""
    import torch
    lens = [40, 17]
    for low in (-float("inf"), torch.finfo(torch.float32).min):
        outs = []
        for fill in (0.0, 1e3, 1e30):
            x = make("bf16", lens, 2, 4, 64, 128, seed=11)
            x["g"][7] = low
            x["g"][42] = low
            x["states"][:2] = fill if fill else x["states"][:2]
            launch(L, form, x)
            torch.cuda.synchronize()
            outs.append((fill, x["o"][7:40].clone(), x["o"][42:57].clone(), x["states"][x["slot_out"].long()].clone()))
        for fill, *got in outs:
            for a, b in zip(outs[0][1:], got):
                assert torch.isfinite(b).all()
                lost = 2.0 ** -17 * fill if form == "prefill" else 0.0
                step = 0.0 if a.dtype == torch.float32 else 2.0 ** -7
                assert float((a.double() - b.double()).abs().max()) <= lost + (step + 1e-5) * float(a.abs().max())
        x = make("bf16", lens, 2, 4, 64, 128, seed=11)
        x["g"][7] = low
        x["g"][42] = low
        check(L, form, x)


@gpu
@pytest.mark.parametrize("form", ["step", "prefill"])
def test_not_a_number_stays_in_its_sequence_and_head(L, form):
    import torch
    x = make("bf16", [20, 19, 21], 2, 4, 64, 128, seed=13)
    y = make("bf16", [20, 19, 21], 2, 4, 64, 128, seed=13)
    x["v"][25, 128:256] = float("nan")                          # sequence 1, value head 1
    x["k"][62] = x["q"][62] = x["v"][62] = float("nan")         # a row behind the last sequence
    launch(L, form, x)
    launch(L, form, y)
    torch.cuda.synchronize()
    bad = torch.zeros(x["rows"], 4, dtype=torch.bool, device="cuda")
    bad[25:39, 1] = True
    assert torch.isnan(x["o"][bad].float()).all()
    assert torch.equal(x["o"][~bad], y["o"][~bad])
    sx, sy = (z["states"][z["slot_out"].long()] for z in (x, y))
    keep = torch.ones(3, 4, dtype=torch.bool, device="cuda")
    keep[1, 1] = False
    assert torch.equal(sx[keep], sy[keep])


@gpu
@pytest.mark.parametrize("form", ["step", "prefill"])
@pytest.mark.parametrize("name", ["q", "k", "v", "g", "beta"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_bad_token_does_not_reach_the_tokens_before_it(L, form, name, bad):
    """The same bits, but in the bad token's own chunk of the prefill form: the powers of two that scale its pieces follow the largest
    numbers of the chunk, the bad token's among them; at either scale the pieces hold 22 bits or 2^-32 of the largest, so that an output
    there may move by 2^-20 of what enters it and then round the other way (one step, 2^-7)."""
    import torch
    x, y = make("bf16", [20, 45, 21], 2, 4, 64, 128, seed=13), make("bf16", [20, 45, 21], 2, 4, 64, 128, seed=13)
    x[name][20 + 23] = bad                                      # sequence 1, all heads
    launch(L, form, x)
    launch(L, form, y)
    torch.cuda.synchronize()
    keep = torch.ones(x["rows"], dtype=torch.bool, device="cuda")
    keep[43:65] = False
    if form == "prefill":
        keep[20:43] = False                                     # a chunk of 64 tokens holds the whole sequence
        a, b = x["o"][20:43].double(), y["o"][20:43].double()
        assert float(((a - b).abs() - 2.0 ** -7 * b.abs()).max()) <= 2.0 ** -20 * float(y["o"][20:65].double().abs().max())
    assert torch.equal(x["o"][keep], y["o"][keep])
    if name == "q":                                             # nothing but its own output
        keep[44:65] = True
        assert torch.equal(x["o"][keep], y["o"][keep])
    assert not torch.isfinite(x["o"][43].float()).all()
    sx, sy = (z["states"][z["slot_out"].long()] for z in (x, y))
    assert torch.equal(sx[[0, 2]], sy[[0, 2]]) and (name == "q") == bool(torch.equal(sx[1], sy[1]))


@gpu
@pytest.mark.parametrize("form", ["step", "prefill"])
def test_a_sequence_gives_the_same_bits_whatever_is_beside_it(L, form):
    """Next to others, and where all others of the call are empty (the prefill form takes its chunks and segments by the call's counts, so
    those stay)."""
    import torch
    for lens in ([18, 1, 33, 0, 16, 47] * 9, [200, 64, 333, 0, 100, 129] * 9):
        x = make("bf16", lens, 2, 4, 128, 128, seed=21)
        launch(L, form, x)
        torch.cuda.synchronize()
        starts = np.concatenate([[0], np.cumsum(lens)])
        for n in (0, 2, 5, 53):
            y = make("bf16", lens, 2, 4, 128, 128, seed=21)
            alone = np.full(len(lens) + 1, starts[n + 1], np.int32)
            alone[:n + 1] = starts[n]
            y["seq_start"] = torch.from_numpy(alone).cuda()
            launch(L, form, y)
            torch.cuda.synchronize()
            assert torch.equal(x["o"][starts[n]:starts[n + 1]], y["o"][starts[n]:starts[n + 1]])
            s = int(y["slot_out"][n])
            assert torch.equal(x["states"][s], y["states"][s])


@gpu
@pytest.mark.parametrize("form", ["step", "prefill"])
def test_captured_replayed_and_on_two_streams(L, form):
    """A captured call replays on new contents of its buffers; two calls with their own buffers run side by side."""
    import torch
    x = make("bf16", [5, 0, 18], 2, 4, 64, 128, seed=31)
    launch(L, form, x)                                          # sizes the workspace outside the capture
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        launch(L, form, x)
    y = make("bf16", [5, 0, 18], 2, 4, 64, 128, seed=32)
    for name in ("q", "k", "v", "g", "beta", "states", "slot_out"):
        x[name].copy_(y[name])
    graph.replay()
    launch(L, form, y)
    torch.cuda.synchronize()
    assert torch.equal(x["o"], y["o"]) and torch.equal(x["states"], y["states"])
    a, b = make("bf16", [64] * 8, 2, 4, 64, 128, seed=41), make("bf16", [64] * 8, 2, 4, 64, 128, seed=42)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        launch(L, form, a, stream=s1)
        launch(L, form, b, stream=s2)
    torch.cuda.synchronize()
    for z, seed in ((a, 41), (b, 42)):
        w = make("bf16", [64] * 8, 2, 4, 64, 128, seed=seed)
        launch(L, form, w)
        torch.cuda.synchronize()
        assert torch.equal(z["o"], w["o"])


@gpu
@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("dk", [64, 128])
def test_calls_behind_one_another_share_states_and_workspace(L, kind, dk):
    """Calls of all forms in turn, each from the states that the one before left and in one workspace: the same bits queued at once,
    captured and replayed, or with a pause behind each."""
    import torch
    hv, dv, n = 4, 128, 3
    shapes = [[1000, 130, 700], [3, 17, 0], [65, 64, 130], [1, 1, 1], [9000, 20, 3000], [40, 30, 33], [300, 2, 1]]
    calls = [make(kind, lens, 2, hv, dk, dv, seed=90 + i) for i, lens in enumerate(shapes)]
    room = max(L.shvk_gdn_prefill_workspace_bytes(C.byref(args(x))) for x in calls)
    ws = torch.empty(room, dtype=torch.uint8, device="cuda")
    states = calls[0]["states"][:n].clone()
    slots = torch.arange(n, device="cuda", dtype=torch.int32)
    for x in calls:
        x["states"], x["n_slots"], x["slot_in"], x["slot_out"] = states, n, slots, slots
    first = states.clone()

    def run(pause, stream):
        for i, x in enumerate(calls):
            a = args(x)
            rc = L.shvk_gdn_step(C.byref(a), stream) if i in (3, 6) else L.shvk_gdn_prefill(C.byref(a), ws.data_ptr(), room, stream)
            assert rc == 0
            if pause:
                torch.cuda.synchronize()

    def result():
        torch.cuda.synchronize()
        got = [states.clone()] + [x["o"].clone() for x in calls]
        states.copy_(first)
        for x in calls:
            x["o"].fill_(7.0)
        torch.cuda.synchronize()
        return got
    run(True, torch.cuda.current_stream().cuda_stream)
    want = result()
    for _ in range(5):
        run(False, torch.cuda.current_stream().cuda_stream)
        assert all(torch.equal(g, w) for g, w in zip(result(), want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(False, torch.cuda.current_stream().cuda_stream)
    result()
    for _ in range(3):
        graph.replay()
        assert all(torch.equal(g, w) for g, w in zip(result(), want))


@gpu
@pytest.mark.parametrize("form", ["step", "prefill", "long"])
@pytest.mark.parametrize("before", ["copy", "fill", "join", "nothing"])
def test_what_a_call_may_stand_behind(L, form, before):
    """Behind a copy, a fill, two streams that meet, or first of all; queued and in a graph: its inputs are the ones written there."""
    import torch
    lens = [9000, 700] if form == "long" else [70, 0, 130]
    x = make("bf16", lens, 2, 4, 128, 128, seed=17)
    form = "prefill" if form == "long" else form
    launch(L, form, x)
    torch.cuda.synchronize()
    states = x["states"].clone()
    names = ("v", "seq_start", "states") if before != "fill" else ("states",)
    good = {name: x[name].clone() for name in names}
    good["states"] = torch.zeros_like(states) if before == "fill" else make("bf16", lens, 2, 4, 128, 128, seed=17)["states"]
    side, fork, joined = torch.cuda.Stream(), torch.cuda.Event(), torch.cuda.Event()

    def run():
        main = torch.cuda.current_stream()
        if before == "join":
            fork.record(main)
            side.wait_event(fork)
            with torch.cuda.stream(side):
                x["v"].copy_(good["v"])
                x["states"].copy_(good["states"])
                joined.record(side)
            x["seq_start"].copy_(good["seq_start"])
            main.wait_event(joined)
        elif before == "fill":
            x["states"].zero_()
        elif before == "copy":
            for name in names:
                x[name].copy_(good[name])
        launch(L, form, x, stream=main)

    def spoil():
        x["o"].fill_(7.0)
        if before in ("copy", "join"):
            x["v"].fill_(1.0)
            x["seq_start"].zero_()
        if before != "nothing":
            x["states"].fill_(3.0)
        else:
            x["states"].copy_(good["states"])
        torch.cuda.synchronize()
    spoil()
    if before in ("copy", "join"):                              # the answer: everything in its place, with a pause in front
        for name in names:
            x[name].copy_(good[name])
    elif before == "fill":
        x["states"].zero_()
    torch.cuda.synchronize()
    launch(L, form, x)
    torch.cuda.synchronize()
    want = (x["o"].clone(), x["states"].clone())
    for _ in range(3):
        spoil()
        run()
        torch.cuda.synchronize()
        assert torch.equal(x["o"], want[0]) and torch.equal(x["states"], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for _ in range(3):
        spoil()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(x["o"], want[0]) and torch.equal(x["states"], want[1])


@gpu
@pytest.mark.parametrize("layer_type", ["bf16", "fp16"])
def test_a_layer_in_service(L, layer_type):
    """The operators as a layer runs them: a prompt by the chunked form, the gated norm over each head's values, then the residual sum and
    the next block's norm; then two more tokens by the step form and the same norms.  Against the formulas in float64 on the same inputs,
    each operator's outputs taken as the next one's inputs (its own tests bound it on those)."""
    import torch
    t = {"bf16": torch.bfloat16, "fp16": torch.float16}[layer_type]
    hv, dv, d = 4, 128, 512
    lens = [70, 200, 1]
    x = make(layer_type, lens, 2, hv, 128, dv, seed=71, tail=0)
    gen = torch.Generator(device="cuda").manual_seed(72)
    rn = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    o_w, next_w = 1 + 0.2 * rn(dv), 1 + 0.2 * rn(d)
    code, s = CODES[layer_type], torch.cuda.current_stream().cuda_stream

    def norms(o, rows):
        """(gated heads, residual stream, normalised rows) by the calls, and checked."""
        gate, h = rn(rows, hv * dv).to(t), 3 * rn(rows, d)
        on, xn, h_out = torch.empty(rows, hv * dv, device="cuda", dtype=t), torch.empty(rows, d, device="cuda", dtype=t), h.clone()
        a = binding.BlockNormArgs(rows=rows, heads=hv, D=dv, x=o.data_ptr(), ldx=hv * dv, x_dtype=code, post_w=o_w.data_ptr(), gate=gate.data_ptr(),
                                  ldgate=hv * dv, gate_dtype=code, gate_act=1, scale=1.0, h_out=on.data_ptr(), ldh_out=hv * dv, h_dtype=code, eps=1e-6)
        assert L.shvk_block_norm(C.byref(a), s) == 0
        b = binding.BlockNormArgs(rows=rows, heads=1, D=d, x=on.data_ptr(), ldx=d, x_dtype=code, scale=0.7, h_in=h_out.data_ptr(), ldh_in=d,
                                  h_out=h_out.data_ptr(), ldh_out=d, h_dtype=0, pre_w=next_w.data_ptr(), xn=xn.data_ptr(), ldxn=d, xn_dtype=code, eps=1e-6)
        assert L.shvk_block_norm(C.byref(b), s) == 0
        o64, g64 = o.double().view(rows, hv, dv), gate.double().view(rows, hv, dv)
        want = o64 / (o64.square().mean(-1, keepdim=True) + 1e-6).sqrt() * o_w.double() * g64 * torch.sigmoid(g64)
        half, err = torch.finfo(t).eps / 2, 128 * 2.0 ** -24
        assert float(((on.double().view_as(want) - want).abs() - (half + err) * want.abs() - 2.0 ** -25).max()) <= 0
        want_h = h.double() + on.double() * float(np.float32(0.7))
        assert float(((h_out.double() - want_h).abs() - err * (h.double().abs() + on.double().abs())).max()) <= 0
        z = h_out.double()
        want_n = z / (z.square().mean(-1, keepdim=True) + 1e-6).sqrt() * next_w.double()
        assert float(((xn.double() - want_n).abs() - (half + 2 * err) * want_n.abs() - err * 4).max()) <= 0
    check(L, "prefill", x)
    norms(x["o"], sum(lens))
    for token in range(2):
        y = make(layer_type, [1, 1, 1], 2, hv, 128, dv, seed=73 + token, tail=0)
        y["states"], y["n_slots"], y["slot_in"], y["slot_out"] = x["states"], x["n_slots"], x["slot_out"], x["slot_out"]
        check(L, "step", y)
        norms(y["o"], 3)


@gpu
def test_waits_that_run_out_end_the_call(L):
    """Nothing is copied for the first chunks: every role gives up in turn, the status word says so, and the next call is right."""
    import subprocess
    import sys
    code = """
import ctypes as C, torch
from tests import test_gdn_seq as T
from shield_sisa_b200 import binding
L = binding.load_library(True)
x = T.make("bf16", [200, 130], 2, 4, 128, 128, seed=3)
T.launch(L, "prefill", x)
torch.cuda.synchronize()
status = C.c_int(-1)
assert L.shvk_gdn_prefill_status(C.byref(status)) == 0 and status.value == 0
a = T.args(x)
assert L.shvk_gdn_prefill_starved(C.byref(a), x["ws"].data_ptr(), x["ws"].numel(), 256, torch.cuda.current_stream().cuda_stream) == 0
torch.cuda.synchronize()
assert L.shvk_gdn_prefill_status(C.byref(status)) == 0 and status.value > 0
T.check(L, "prefill", T.make("bf16", [200, 130], 2, 4, 128, 128, seed=4))
print("ended with status", status.value)
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120, cwd=str(__import__("tests.helpers", fromlist=["ROOT"]).ROOT))
    assert r.returncode == 0, r.stderr[-2000:]                 # in a process of its own: the word stays set
    assert "ended with status" in r.stdout


def test_status_fetch_refuses_no_place(L):
    assert L.shvk_gdn_prefill_status_fetch_async(None, None) == INVALID


@gpu
def test_status_word_is_read_and_cleared_behind_the_work(L):
    """The word of a call whose waits ran out, fetched and cleared on the call's stream; the next call leaves it clear."""
    import subprocess
    import sys
    code = """
import ctypes as C, torch
from tests import test_gdn_seq as T
from shield_sisa_b200 import binding
L = binding.load_library(True)
x = T.make("fp16", [200, 130], 2, 4, 64, 128, seed=3)
T.launch(L, "prefill", x)
word = torch.full((3,), -1, dtype=torch.int32).pin_memory()
stream = torch.cuda.Stream()
torch.cuda.synchronize()
a = T.args(x)
assert L.shvk_gdn_prefill_starved(C.byref(a), x["ws"].data_ptr(), x["ws"].numel(), 256, stream.cuda_stream) == 0
assert L.shvk_gdn_prefill_status_fetch_async(word.data_ptr(), stream.cuda_stream) == 0
assert L.shvk_gdn_prefill_status_clear_async(stream.cuda_stream) == 0
assert L.shvk_gdn_prefill_status_fetch_async(word.data_ptr() + 4, stream.cuda_stream) == 0
stream.synchronize()
T.check(L, "prefill", T.make("fp16", [200, 130], 2, 4, 64, 128, seed=4))
assert L.shvk_gdn_prefill_status_fetch_async(word.data_ptr() + 8, stream.cuda_stream) == 0
stream.synchronize()
print("words", word[0].item() > 0, word[1].item(), word[2].item())
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120, cwd=str(__import__("tests.helpers", fromlist=["ROOT"]).ROOT))
    assert r.returncode == 0, r.stderr[-2000:]
    assert "words True 0 0" in r.stdout


@gpu
def test_slots_past_two_gigabytes(L):
    """A pool whose last slots lie beyond 2^31 values."""
    import torch
    hv, dk, dv = 16, 128, 256
    slots = (1 << 31) // (hv * dk * dv) + 3
    x = make("bf16", [1, 2], 2, hv, dk, dv, seed=51)
    small = x["states"][:2].clone()
    x["states"] = torch.empty(slots, hv, dk, dv, device="cuda")
    x["n_slots"] = slots
    x["states"][slots - 2:] = small
    x["slot_in"] = torch.tensor([slots - 2, -1], device="cuda", dtype=torch.int32)
    x["slot_out"] = torch.tensor([slots - 1, slots - 3], device="cuda", dtype=torch.int32)
    want, states, _ = rule(x, [small[0], torch.zeros_like(small[0])])
    launch(L, "step", x)
    torch.cuda.synchronize()
    for s, ref in ((slots - 1, states[0]), (slots - 3, states[1])):
        assert float((x["states"][s].double() - ref).abs().max()) < 1e-5 * float(ref.abs().max())
    assert torch.equal(x["states"][slots - 2], small[0])
    del x
    torch.cuda.empty_cache()


def form_of(L, x):
    """Chunks of how many tokens the prefill takes this call in: those of 16 need 2,448 bytes for each chunk and value head, those of 64
    another size."""
    need = L.shvk_gdn_prefill_workspace_bytes(C.byref(args(x)))
    return 16 if need == (x["rows"] // 16 + x["n"] + 1) * x["hv"] * 2448 else 64


def assert_float32_outputs(x, want):
    """The outputs are the rule's to float32's accuracy before they are rounded, in either type (check allows bf16 outputs single pieces of
    eleven bits on their way, which they no longer come from): few of them are another value of the type than the
    float64 ones' rounding.  An error e moves an output over a tie with a probability of 2 e / step, a step is at least eps / 2 of the
    value, and the mean of rms / |value| is some 4 (a normal value's, down to a thousandth of the rms).  With e within 2^-19 of the rms
    (the state's error is held to 1e-6 of its norm, half of that), that is 16 x 2^-19 / eps of the outputs: 0.4 % for bf16, 3 % for fp16.
    (Pieces of eleven bits, e of 2^-12, move 16 x 2^-12 / 2^-7 = 50 % at most, and some 5 % where they are off by chance.)"""
    import torch
    total = sum(x["lens"])
    wrong = float((x["o"][:total] != want[:total].to(x["o"].dtype)).double().mean())
    print(f"outputs that are not the float64 ones' rounding: {100 * wrong:.3f} %")
    assert wrong <= 16 * 2.0 ** -19 / torch.finfo(x["o"].dtype).eps


@gpu
@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("form,layout,lens", [(16, (2, 6, 128, 128), [48, 0, 17, 33] * 5), (16, (6, 6, 64, 64), [100] * 30),
                                              (16, (3, 3, 64, 32), [300, 129]), (16, (1, 1, 128, 96), [500]),
                                              (64, (2, 6, 128, 128), [333, 64, 0, 190]), (64, (6, 6, 64, 128), [321]),
                                              (64, (2, 2, 128, 256), [200, 77]), (64, (2, 4, 64, 192), [140, 300]),
                                              (64, (1, 4, 64, 64), [150, 260]), (64, (1, 1, 128, 128), [3000])], ids=str)
def test_prefill_outputs_are_float32_before_they_are_rounded(L, kind, form, layout, lens):
    import torch
    x = make(kind, lens, *layout, seed=len(lens) + layout[2])
    assert form_of(L, x) == form
    want, _, _ = rule(x, first_states(x))
    check(L, "prefill", x)
    assert_float32_outputs(x, want)
    first, states = x["o"].clone(), x["states"].clone()          # whatever o's rows held before
    x["o"][:sum(lens)] = torch.nan
    launch(L, "prefill", x)
    torch.cuda.synchronize()
    assert torch.equal(x["o"], first) and torch.equal(x["states"], states)


# ---------------------------------------------------------------------------------------------- each form of the prefill at its edges
SHORT = [(16, (2, 4, 64, 128), [20, 0, 33]), (16, (2, 4, 128, 128), [70, 0, 26])]
FULL = [(64, (2, 4, 128, 128), [200, 0, 330]), (64, (2, 4, 64, 128), [300, 0, 260])]
SEGMENTS = (64, (1, 2, 128, 128), [3900, 0, 5000])


def of_form(L, case, kind="bf16", **kw):
    form, layout, lens = case
    x = make(kind, lens, *layout, **kw)
    assert form_of(L, x) == form
    return x


@gpu
@pytest.mark.parametrize("case", SHORT + FULL, ids=str)
@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("name", list(slot_cases()))
def test_slots_in_each_form(L, case, kind, name):
    import torch
    s = tuple(None if v is None else torch.tensor(v, device="cuda", dtype=torch.int32) for v in slot_cases()[name])
    x = of_form(L, case, kind, seed=3, slots=s)
    want, _, _ = rule(x, first_states(x))
    check(L, "prefill", x)
    assert_float32_outputs(x, want)
    if name == "none":                                          # no pool at all
        got, a = x["o"].clone(), args(x)
        a.states, a.n_slots = None, 0
        assert call(L, "prefill", a, x["ws"].data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        assert torch.equal(x["o"], got)


@gpu
@pytest.mark.parametrize("name", ["in_place", "new", "not_kept", "outside"])
def test_slots_of_sequences_in_segments(L, name):
    import torch
    s = tuple(torch.tensor(v, device="cuda", dtype=torch.int32) for v in slot_cases()[name])
    x = of_form(L, SEGMENTS, seed=4, slots=s)
    x["g"] *= 0.1
    assert L.shvk_gdn_prefill_workspace_bytes(C.byref(args(x))) > 16912 * (x["rows"] // 64 + x["n"]) * x["hv"]      # states of segments
    check(L, "prefill", x)


@gpu
@pytest.mark.parametrize("case", FULL, ids=str)
@pytest.mark.parametrize("kind", ["bf16", "fp16"])
def test_bounds_that_are_no_bounds_in_chunks_of_64(L, case, kind):
    """The first sequence is well described, the others have starts outside the rows."""
    import torch
    x, y = (of_form(L, case, kind, seed=9, tail=0) for _ in range(2))
    rows, first = x["rows"], case[2][0]
    x["seq_start"] = torch.tensor([0, first, -9, 1 << 30], device="cuda", dtype=torch.int32)      # its rows; none; all
    y["seq_start"] = torch.tensor([0, first, first, first], device="cuda", dtype=torch.int32)
    guards = [torch.full((rows + 256,) + x["o"].shape[1:], 7.0, device="cuda").to(x["o"].dtype) for _ in range(2)]
    for z, g in zip((x, y), guards):
        z["o"] = g[:rows]
    pool = x["states"].clone()
    launch(L, "prefill", x)
    launch(L, "prefill", y)
    torch.cuda.synchronize()
    slot = int(x["slot_out"][0])
    assert torch.equal(x["states"][slot], y["states"][slot]) and not torch.equal(pool[slot], x["states"][slot])
    assert torch.equal(x["states"][2 * x["n"]], pool[2 * x["n"]]) and torch.equal(x["states"][:x["n"]], pool[:x["n"]])
    assert all(torch.equal(g[rows:], torch.full_like(g[rows:], 7.0)) for g in guards)


@gpu
@pytest.mark.parametrize("form,layout,lens,at,lost", [(16, (2, 4, 64, 128), [40, 17], 7, 2.0 ** -24), (64, (2, 4, 64, 128), [160, 150], 70, 2.0 ** -17),
                                                      (64, (2, 4, 128, 128), [160, 150], 70, 2.0 ** -16)], ids=str)
@pytest.mark.parametrize("low", [-float("inf"), -3.4028234663852886e38])
def test_a_decay_to_nothing_in_each_form(L, form, layout, lens, at, lost, low):
    """As test_a_decay_to_nothing_forgets_everything has it, with each form's bound: chunks of 16 hold W to 2^-35 of a column's largest, so
    16 x 8 x 2^-35 x 16 = 2^-24 of the fill; of 64, 64 x 8 x 2^-32 x 64 = 2^-17, with 128 keys (|k|_1 <= 11.4) 2^-16 at most."""
    import torch
    outs = []
    for fill in (0.0, 1e3, 1e30):
        x = of_form(L, (form, layout, lens), seed=11)
        x["g"][at] = low
        x["g"][lens[0] + 2] = low
        x["states"][:2] = fill if fill else x["states"][:2]
        launch(L, "prefill", x)
        torch.cuda.synchronize()
        outs.append((fill, x["o"][at:lens[0]].clone(), x["o"][lens[0] + 2:sum(lens)].clone(), x["states"][x["slot_out"].long()].clone()))
    for fill, *got in outs:
        for a, b in zip(outs[0][1:], got):
            assert torch.isfinite(b).all()
            step = 0.0 if a.dtype == torch.float32 else 2.0 ** -7
            assert float((a.double() - b.double()).abs().max()) <= lost * fill + (step + 1e-5) * float(a.abs().max())
    x = of_form(L, (form, layout, lens), seed=11)
    x["g"][at] = low
    x["g"][lens[0] + 2] = low
    want, _, _ = rule(x, first_states(x))
    check(L, "prefill", x)
    assert_float32_outputs(x, want)


@gpu
@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("dk", [64, 128])
def test_not_a_number_stays_in_its_sequence_and_head_in_chunks_of_64(L, kind, dk):
    """In one head's values of a sequence, in rows behind the last sequence (which a chunk's copies may bring in), and all over a sequence
    beside others."""
    import torch
    case = (64, (2, 4, dk, 128), [150, 200, 130])
    x, y = (of_form(L, case, kind, seed=13, tail=70) for _ in range(2))
    x["v"][170, 128:256] = float("nan")                         # sequence 1, value head 1
    for name in ("q", "k", "v", "g", "beta"):
        x[name][480:] = float("nan")
    launch(L, "prefill", x)
    launch(L, "prefill", y)
    torch.cuda.synchronize()
    bad = torch.zeros(x["rows"], 4, dtype=torch.bool, device="cuda")
    bad[170:350, 1] = True
    assert torch.isnan(x["o"][bad].float()).all()
    near = torch.zeros_like(bad)
    near[150:170, 1] = True                                     # the bad token's own chunk (see the test of bad tokens)
    assert torch.equal(x["o"][~bad & ~near], y["o"][~bad & ~near])
    assert torch.isfinite(x["o"][near].float()).all()
    sx, sy = (z["states"][z["slot_out"].long()] for z in (x, y))
    keep = torch.ones(3, 4, dtype=torch.bool, device="cuda")
    keep[1, 1] = False
    assert torch.equal(sx[keep], sy[keep]) and torch.isnan(sx[1, 1]).all()
    for name in ("q", "k", "v", "g", "beta"):                   # a whole sequence
        x[name][150:350] = float("nan")
    launch(L, "prefill", x)
    torch.cuda.synchronize()
    keep = torch.ones(x["rows"], dtype=torch.bool, device="cuda")
    keep[150:350] = False
    assert torch.equal(x["o"][keep], y["o"][keep]) and torch.isnan(x["o"][150:350].float()).all()
    sx = x["states"][x["slot_out"].long()]
    assert torch.equal(sx[[0, 2]], sy[[0, 2]]) and torch.isnan(sx[1]).all()


@gpu
@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("case,bad_at", [((16, (2, 4, 64, 128), [20, 45, 21]), 23), ((64, (2, 4, 64, 128), [150, 200, 130]), 100),
                                         ((64, (2, 4, 128, 128), [150, 200, 130]), 100)], ids=str)
@pytest.mark.parametrize("name", ["q", "k", "v", "g", "beta"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_bad_token_in_each_form(L, kind, case, bad_at, name, bad):
    """As test_a_bad_token_does_not_reach_the_tokens_before_it has it: other bits in the bad token's own chunk alone, and there by 2^-20 of
    what enters an output and one step of its type."""
    import torch
    x, y = (of_form(L, case, kind, seed=13) for _ in range(2))
    (a0, a1, _), chunk = case[2], case[0]
    token, begin, end = a0 + bad_at, a0 + bad_at // chunk * chunk, a0 + a1
    x[name][token] = bad
    launch(L, "prefill", x)
    launch(L, "prefill", y)
    torch.cuda.synchronize()
    keep = torch.ones(x["rows"], dtype=torch.bool, device="cuda")
    keep[begin:end] = False
    assert torch.equal(x["o"][keep], y["o"][keep])
    a, b = x["o"][begin:token].double(), y["o"][begin:token].double()
    assert token > begin and float(((a - b).abs() - torch.finfo(x["o"].dtype).eps * b.abs()).max()) <= 2.0 ** -20 * float(y["o"][a0:end].double().abs().max())
    assert not torch.isfinite(x["o"][token].float()).all()
    if name == "q":                                             # nothing but its own output
        assert torch.equal(x["o"][token + 1:end], y["o"][token + 1:end])
    sx, sy = (z["states"][z["slot_out"].long()] for z in (x, y))
    assert torch.equal(sx[[0, 2]], sy[[0, 2]]) and (name == "q") == bool(torch.equal(sx[1], sy[1]))


@gpu
@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("dk", [64, 128])
@pytest.mark.parametrize("unit", [False, True])
def test_chunks_of_64_on_slices_of_one_row(L, kind, dk, unit):
    """q, k and v side by side in rows that are wider than they are, outputs in rows with room between them."""
    import torch
    x = of_form(L, (64, (2, 4, dk, 128), [300, 5, 130]), kind, seed=5, fused=True, unit=unit)
    wide = torch.full((x["rows"], 6, 128), 7.0, device="cuda").to(x["o"].dtype)
    x["o"] = wide[:, 1:5]
    want, _, _ = rule(x, first_states(x))
    check(L, "prefill", x)
    assert_float32_outputs(x, want)
    assert torch.equal(wide[:, [0, 5]], torch.full_like(wide[:, [0, 5]], 7.0))


@gpu
@pytest.mark.parametrize("case", FULL + [SEGMENTS], ids=str)
@pytest.mark.parametrize("kind", ["bf16", "fp16"])
def test_chunks_of_64_captured_replayed_and_on_two_streams(L, case, kind):
    import torch
    x, y = of_form(L, case, kind, seed=31), of_form(L, case, kind, seed=32)
    launch(L, "prefill", x)                                     # sizes the workspace outside the capture
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        launch(L, "prefill", x)
    for name in ("q", "k", "v", "g", "beta", "states", "slot_out"):
        x[name].copy_(y[name])
    graph.replay()
    launch(L, "prefill", y)
    torch.cuda.synchronize()
    assert torch.equal(x["o"], y["o"]) and torch.equal(x["states"], y["states"])
    calls = [of_form(L, case, kind, seed=41 + i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(3):
        for z, s in zip(calls, streams):
            launch(L, "prefill", z, stream=s)
    torch.cuda.synchronize()
    for i, z in enumerate(calls):
        w = of_form(L, case, kind, seed=41 + i)
        launch(L, "prefill", w)
        torch.cuda.synchronize()
        assert torch.equal(z["o"], w["o"]) and torch.equal(z["states"], w["states"])


@gpu
@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("dk", [64, 128])
def test_steps_continue_what_chunks_of_64_left(L, kind, dk):
    """A prompt in two calls of the chunked form, the second from where the first stopped, then tokens in place, against one walk of all."""
    import torch
    layout, cuts = (2, 4, dk, 128), [(200, 130), (150, 140), (141, 300)]
    new = 3
    lens = [a + b + new for a, b in cuts]
    whole = make(kind, lens, *layout, seed=23, tail=0)
    want, states, _ = rule(whole, first_states(whole))
    starts = np.concatenate([[0], np.cumsum(lens)])
    half = torch.finfo(whole["o"].dtype).eps / 2
    factor = (dk + 24 * max(lens)) * 2.0 ** -24
    big = max(float(s.norm(dim=1).max()) for s in states) + float(want.abs().max()) + float(whole["states"].norm(dim=2).max())
    done = [0, 0, 0]
    for step, size in enumerate([[a for a, _ in cuts], [b for _, b in cuts]] + [[1, 1, 1]] * new):
        pick = torch.tensor([starts[i] + done[i] + j for i in range(3) for j in range(size[i])], device="cuda")
        x = dict(whole)
        x.pop("ws", None)
        for name in ("q", "k", "v", "g", "beta"):
            x[name] = whole[name][pick].contiguous()
        x["rows"], x["lens"] = len(pick), size
        x["o"] = torch.full((len(pick), 4, 128), 7.0, device="cuda").to(whole["o"].dtype)
        x["seq_start"] = torch.from_numpy(np.concatenate([[0], np.cumsum(size)]).astype(np.int32)).cuda()
        if step:
            x["slot_in"] = whole["slot_out"]
        if step < 2:
            assert form_of(L, x) == 64
        launch(L, "prefill" if step < 2 else "step", x)
        torch.cuda.synchronize()
        ref = want[pick]
        assert float(((x["o"].double() - ref).abs() - half * ref.abs()).max()) <= factor * big + (2.0 ** -25 if kind == "fp16" else 0.0)
        done = [d + s for d, s in zip(done, size)]
    for i in range(3):
        got = whole["states"][int(whole["slot_out"][i])].double()
        assert float((got - states[i]).abs().max()) <= factor * max(float(states[i].norm(dim=1).max()), big)


@gpu
@pytest.mark.parametrize("form", ["step", "prefill"])
def test_no_rows_at_all_copy_the_states(L, form):
    """Sequences in a call without a single row: states go from slot to slot, or start from zero; no array of rows is there."""
    import torch
    for dk, slots in ((64, ([2, 0, -1], [4, 5, 6])), (128, ([1, 1, 0], [3, -1, 0])), (64, (None, [0, 1, 2]))):
        s = tuple(None if v is None else torch.tensor(v, device="cuda", dtype=torch.int32) for v in slots)
        x = make("bf16", [0, 0, 0], 2, 4, dk, 128, seed=5, tail=0, slots=s)
        first, pool = first_states(x), x["states"].clone()
        a = args(x)
        a.q = a.k = a.v = a.g = a.beta = a.o = None
        need = L.shvk_gdn_prefill_workspace_bytes(C.byref(a))
        ws = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
        assert call(L, form, a, ws.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        for n, out in enumerate(slots[1]):
            if out >= 0:
                pool[out] = first[n]
        assert torch.equal(x["states"], pool)


@gpu
@pytest.mark.parametrize("form,layout,lens", [("step", (2, 4, 64, 128), [3, 0, 2]), (16, (2, 4, 128, 128), [40, 0, 26]), (64, (2, 4, 128, 128), [200, 0, 330])], ids=str)
def test_rows_past_two_gigabytes(L, form, layout, lens):
    """Rows so far apart that the last ones lie beyond 2^31 values of their arrays."""
    import torch
    x = make("bf16", lens, *layout, seed=53)
    y = dict(x)
    y["states"] = x["states"].clone()
    rows = x["rows"]
    pitch = ((1 << 31) // (rows - 5) // 8 + 1) * 8
    flat = torch.empty(rows * pitch, device="cuda", dtype=torch.bfloat16)
    big = flat.view(rows, pitch)
    at = 0
    for name in ("q", "k", "v"):                                # one behind the other in rows of one array
        w = x[name].shape[1]
        big[:, at:at + w] = x[name]
        y[name] = big[:, at:at + w]
        at += w
    y["o"] = big[:, at:at + layout[1] * layout[3]].unflatten(1, (layout[1], layout[3]))
    y["o"].fill_(7.0)
    assert (rows - 4) * pitch > 1 << 31
    if form != "step":
        assert form_of(L, x) == form and form_of(L, y) == form
    for z in (x, y):
        launch(L, "step" if form == "step" else "prefill", z)
    torch.cuda.synchronize()
    assert torch.equal(x["o"], y["o"]) and torch.equal(x["states"], y["states"]) and torch.isfinite(x["o"].float()).all()
    del x, y, big, flat
    torch.cuda.empty_cache()
