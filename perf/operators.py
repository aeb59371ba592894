"""Operators of a gated-delta-rule layer that keeps its state between calls, as cases that can be timed and compared.

Three operators, each a call of the launch layer (include/shv_seq_kernels.h) that works on a user's device buffers:

  step      shvk_gdn_step: the gated delta rule, recurrent, one or a few new tokens of every live sequence, states read
            from a pool's slots and written back to slots
  prefill   shvk_gdn_prefill: the same rule in chunks, over packed sequences of any lengths, states taken from and left in
            the pool
  norm      shvk_block_norm: what stands between two blocks of a layer in one pass over the rows: RMS norm of a block's
            output, its gate and scale, the residual sum, and the RMS norm in front of the next block; also, without a
            residual, the gated norm over each head's values that follows the delta rule

A case is run on inputs that look like a trained layer's: keys and queries behind a SiLU, decays -A softplus(.) with rates
A spread over the heads, learning rates sigmoid(.), states of the size that the rule itself leaves.
"""
import ctypes
import random

import torch

own = False

EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CODES = {"fp32": 0, "bf16": 1, "fp16": 2}
SIZES = {"fp32": 4, "bf16": 2, "fp16": 2}


def listed():
    return [
        # one live stream's next token in a layer of the detector's size: nothing but latency
        {"name": "step_1_dk64", "op": "step", "n": 1, "t": 1, "ragged": False, "hk": 6, "hv": 6, "dk": 64, "dv": 128, "type": "bf16"},
        # an odd number of streams, some with a few accepted draft tokens at once and some with none, shared key heads
        {"name": "step_45_ragged", "op": "step", "n": 45, "t": 5, "ragged": True, "hk": 2, "hv": 6, "dk": 128, "dv": 128, "type": "fp16"},
        # the exact tier's stream batch
        {"name": "step_128_fp32", "op": "step", "n": 128, "t": 1, "ragged": False, "hk": 6, "hv": 6, "dk": 64, "dv": 128, "type": "fp32"},
        # a full batch of streams with the wider keys: reading and writing the states is all it does
        {"name": "step_512_dk128", "op": "step", "n": 512, "t": 1, "ragged": False, "hk": 6, "hv": 6, "dk": 128, "dv": 128, "type": "bf16"},
        # one clip's 321 tokens: too few heads to fill the GPU
        {"name": "prefill_1x321_dk64", "op": "prefill", "n": 1, "t": 321, "ragged": False, "hk": 6, "hv": 6, "dk": 64, "dv": 128, "type": "bf16"},
        # prompts of odd lengths packed together, an empty one and one of a single token among them, shared key heads
        {"name": "prefill_37_ragged", "op": "prefill", "n": 37, "t": 1021, "ragged": True, "hk": 2, "hv": 6, "dk": 128, "dv": 128, "type": "fp16"},
        # one long history
        {"name": "prefill_1x16384", "op": "prefill", "n": 1, "t": 16384, "ragged": False, "hk": 6, "hv": 6, "dk": 128, "dv": 128, "type": "bf16"},
        # the long-sequence stress configuration, now with its states
        {"name": "prefill_64x2048", "op": "prefill", "n": 64, "t": 2048, "ragged": False, "hk": 6, "hv": 6, "dk": 128, "dv": 128, "type": "bf16"},
        # one token's row of the detector's width between two blocks
        {"name": "norm_1x384", "op": "norm", "rows": 1, "heads": 1, "d": 384, "type": "bf16", "post": True, "gate": "rows", "act": "silu", "res": "fp32", "pre": True},
        # the gated norm over every head's 128 values behind the delta rule, 64 clips
        {"name": "norm_heads_123264x128", "op": "norm", "rows": 20544, "heads": 6, "d": 128, "type": "bf16", "post": True, "gate": "rows", "act": "silu", "res": "none", "pre": False},
        # the residual stream of 64 clips: a projection's 16-bit output added to fp32 rows, normalised for the next block
        {"name": "norm_20544x384", "op": "norm", "rows": 20544, "heads": 1, "d": 384, "type": "fp16", "post": False, "gate": "none", "act": "none", "res": "fp32", "pre": True},
        # an odd width that no vector load divides, one gate row for all rows (a layer scale), everything on
        {"name": "norm_16384x2047", "op": "norm", "rows": 16384, "heads": 1, "d": 2047, "type": "bf16", "post": True, "gate": "one", "act": "sigmoid", "res": "bf16", "pre": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["step", "prefill", "norm"])
    if op == "norm":
        d = rng.choice([128, 384, 768, 960, 1920, _log(rng, 33, 4096), _log(rng, 33, 4096)])
        heads = rng.choice([1, 1, 1, 6])
        rows = _log(rng, 1, max(1, min(65536, 33_000_000 // (d * heads))))
        kind = rng.choice(["bf16", "fp16"])
        return {"op": op, "rows": rows, "heads": heads, "d": d, "type": kind, "post": rng.random() < 0.7,
                "gate": rng.choice(["none", "rows", "rows", "one"]), "act": rng.choice(["none", "silu", "sigmoid"]),
                "res": rng.choice(["none", "fp32", "fp32", kind]), "pre": rng.random() < 0.7}
    hk, hv = rng.choice([(6, 6), (6, 6), (2, 6), (4, 8), (1, 4)])
    dk, dv = rng.choice([64, 128]), rng.choice([64, 128, 128, 128])
    case = {"op": op, "hk": hk, "hv": hv, "dk": dk, "dv": dv, "ragged": rng.random() < 0.5}
    if op == "step":
        return {**case, "n": _log(rng, 1, max(1, 512 * 6 * 128 * 128 // (hv * dk * 128))), "t": rng.choice([1, 1, 1, 2, 3, 4, 8]),
                "type": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    t = _log(rng, 16, 16384)
    return {**case, "t": t, "n": _log(rng, 1, max(1, 64 * 2048 * 6 // (t * hv))), "type": rng.choice(["bf16", "bf16", "fp16"])}


def _lengths(case):
    """Tokens of each sequence: all the same, or from none to t."""
    n, t = case["n"], case["t"]
    if not case["ragged"]:
        return [t] * n
    rng = random.Random(1000003 * n + 101 * t + case["dk"])
    lens = [rng.randint(0, t) for _ in range(n)]
    lens[0] = t
    if n > 2:
        lens[1], lens[2] = 0, 1
    return lens


def work(case):
    if case["op"] == "norm":
        rows, d, size = case["rows"] * case["heads"], case["d"], SIZES[case["type"]]
        res = SIZES[case["res"]] if case["res"] != "none" else 0
        per = size + (size if case["gate"] == "rows" else 0) + res + (res or size) + (size if case["pre"] else 0)
        return {"bytes": rows * d * per + 4 * d * (case["post"] + case["pre"]), "flops": 12 * rows * d}
    tokens, hk, hv, dk, dv, size = sum(_lengths(case)), case["hk"], case["hv"], case["dk"], case["dv"], SIZES[case["type"]]
    state = case["n"] * hv * dk * dv
    return {"bytes": tokens * ((2 * hk * dk + 2 * hv * dv) * size + 8 * hv) + 8 * state, "flops": 6 * tokens * hv * dk * dv}


class _State:
    pass


def prepare(case, seed):
    s = _State()
    s.case = case
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    kind = TYPES[case["type"]]
    rn = lambda *shape: torch.randn(*shape, device="cuda", generator=gen)  # noqa: E731
    if case["op"] == "norm":
        rows, heads, d = case["rows"], case["heads"], case["d"]
        s.x = (rn(rows, heads * d) * 1.5).to(kind)
        s.gate = None if case["gate"] == "none" else rn(rows if case["gate"] == "rows" else 1, heads * d).to(kind)
        s.post_w = 1 + 0.2 * rn(d) if case["post"] else None
        s.pre_w = 1 + 0.2 * rn(d) if case["pre"] else None
        s.h_in = (rn(rows, heads * d) * 3).to(TYPES[case["res"]]) if case["res"] != "none" else None
        s.h_out = torch.empty(rows, heads * d, device="cuda", dtype=kind if s.h_in is None else s.h_in.dtype)
        s.xn = torch.empty(rows, heads * d, device="cuda", dtype=kind) if case["pre"] else None
        s.scale = 0.5
        return s
    n, hk, hv, dk, dv = (case[k] for k in ("n", "hk", "hv", "dk", "dv"))
    lens = _lengths(case)
    s.lens = lens
    s.tokens = sum(lens) + (3 if case["ragged"] else 0)          # a batch padded behind its last sequence
    starts = [0]
    for x in lens:
        starts.append(starts[-1] + x)
    s.seq_start = torch.tensor(starts, dtype=torch.int32, device="cuda")
    silu = torch.nn.functional.silu
    s.q, s.k = silu(rn(s.tokens, hk, dk)).to(kind), silu(rn(s.tokens, hk, dk)).to(kind)
    s.v = silu(rn(s.tokens, hv, dv)).to(kind)
    rate = torch.exp(torch.linspace(-3.0, 1.5, hv, device="cuda"))
    s.g = -rate * torch.nn.functional.softplus(rn(s.tokens, hv) - 2.0)
    s.beta = torch.sigmoid(rn(s.tokens, hv))
    s.o = torch.zeros(s.tokens, hv, dv, device="cuda", dtype=kind)
    s.scale = dk ** -0.5
    s.pool = torch.zeros(2 * n, hv, dk, dv, device="cuda")       # the states before the call, then those after it
    s.pool[:n] = 0.3 * rn(n, hv, dk, dv)
    s.slot_in = torch.randperm(n, device="cuda", generator=gen).to(torch.int32)
    s.slot_out = n + torch.randperm(n, device="cuda", generator=gen).to(torch.int32)
    s.workspace = None
    if case["op"] == "prefill":                                  # memory that a program keeps, one piece for all its layers
        blocks = s.tokens // 16 + n + 1
        s.workspace = torch.empty(blocks * hv * 8192, dtype=torch.uint8, device="cuda")
    return s


def run(s):
    if own:
        return _norm_own(s) if s.case["op"] == "norm" else _delta_own(s)
    return {"norm": _norm_plain, "step": _step_plain, "prefill": _prefill_plain}[s.case["op"]](s)


# ---------------------------------------------------------------------------------------------- the framework's calls
def _delta_own(s):
    from shield_sisa_b200 import binding

    lib, c = binding.load_library(True), s.case
    hk, hv, dk, dv = c["hk"], c["hv"], c["dk"], c["dv"]
    a = binding.GdnSeqArgs(n_seq=c["n"], HK=hk, HV=hv, DK=dk, DV=dv, dtype=CODES[c["type"]], l2norm=1, scale=s.scale,
                           n_tokens=s.tokens, q=s.q.data_ptr(), ldq=hk * dk, k=s.k.data_ptr(), ldk=hk * dk,
                           v=s.v.data_ptr(), ldv=hv * dv, g=s.g.data_ptr(), beta=s.beta.data_ptr(), ldgb=hv,
                           o=s.o.data_ptr(), ldo=hv * dv, seq_start=s.seq_start.data_ptr(), states=s.pool.data_ptr(),
                           n_slots=2 * c["n"], slot_in=s.slot_in.data_ptr(), slot_out=s.slot_out.data_ptr())
    stream = torch.cuda.current_stream().cuda_stream
    if c["op"] == "step":
        rc = lib.shvk_gdn_step(ctypes.byref(a), stream)
    else:
        rc = lib.shvk_gdn_prefill(ctypes.byref(a), s.workspace.data_ptr(), s.workspace.numel(), stream)
    if rc:
        raise RuntimeError("cudaError %d" % rc)
    return s.o, s.pool[c["n"]:]


def _norm_own(s):
    from shield_sisa_b200 import binding

    lib, c = binding.load_library(True), s.case
    ld = c["heads"] * c["d"]
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    h_type = c["type"] if c["res"] == "none" else c["res"]
    a = binding.BlockNormArgs(rows=c["rows"], heads=c["heads"], D=c["d"], x=ptr(s.x), ldx=ld, x_dtype=CODES[c["type"]],
                              post_w=ptr(s.post_w), gate=ptr(s.gate), ldgate=0 if c["gate"] == "one" else ld,
                              gate_dtype=CODES[c["type"]], gate_act={"none": 0, "silu": 1, "sigmoid": 2}[c["act"]],
                              scale=s.scale, h_in=ptr(s.h_in), ldh_in=ld, h_out=ptr(s.h_out), ldh_out=ld,
                              h_dtype=CODES[h_type], pre_w=ptr(s.pre_w), xn=ptr(s.xn), ldxn=ld, xn_dtype=CODES[c["type"]],
                              eps=EPS)
    rc = lib.shvk_block_norm(ctypes.byref(a), torch.cuda.current_stream().cuda_stream)
    if rc:
        raise RuntimeError("cudaError %d" % rc)
    return [s.h_out] + ([s.xn] if s.xn is not None else [])


# ---------------------------------------------------------------------------------------------- the plain forms
def _rms(x, w):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w


def _norm_plain(s):
    c = s.case
    y = s.x.float().view(c["rows"], c["heads"], c["d"])
    if s.post_w is not None:
        y = _rms(y, s.post_w)
    if s.gate is not None:
        g = s.gate.float().view(-1, c["heads"], c["d"])
        y = y * (g if c["act"] == "none" else torch.sigmoid(g) * (g if c["act"] == "silu" else 1.0))
    h = y * s.scale
    if s.h_in is not None:
        h = s.h_in.float().view_as(h) + h
    out = [h.view(s.h_out.shape).to(s.h_out.dtype)]
    if s.pre_w is not None:
        out.append(_rms(h, s.pre_w).view(s.xn.shape).to(s.xn.dtype))
    return out


def _pad(s, x, t, heads):
    """Packed rows [tokens, heads, ...] as [n, hv, t, ...] in 32 bits, zeros behind each sequence's end, key heads repeated."""
    c = s.case
    at = torch.arange(t, device="cuda")
    start, stop = s.seq_start[:-1].long(), s.seq_start[1:].long()
    here = start[:, None] + at
    live = here < stop[:, None]
    rows = x[torch.where(live, here, 0)].float()
    rows = rows * live.view(live.shape + (1,) * (rows.dim() - 2))
    return rows.transpose(1, 2).repeat_interleave(c["hv"] // heads, 1), here, live


def _padded(s, t):
    """(q, k, v, g, beta) by sequence and value head, q and k normalised, and where their rows come from."""
    c = s.case
    q, here, live = _pad(s, s.q, t, c["hk"])
    k, v = _pad(s, s.k, t, c["hk"])[0], _pad(s, s.v, t, c["hv"])[0]
    g, beta = _pad(s, s.g, t, c["hv"])[0], _pad(s, s.beta, t, c["hv"])[0]
    q = q * torch.rsqrt((q * q).sum(-1, keepdim=True) + EPS) * s.scale
    k = k * torch.rsqrt((k * k).sum(-1, keepdim=True) + EPS)
    return q, k, v, g, beta, here, live


def _packed(s, o, state, here, live):
    """Outputs [n, hv, t, dv] as the call leaves them: packed rows, and the states by slot."""
    out = torch.zeros_like(s.o)
    out[here[live]] = o.transpose(1, 2)[live].to(out.dtype)
    after = torch.empty_like(state)
    after[s.slot_out.long() - s.case["n"]] = state
    return out, after


def _step_plain(s):
    """The rule itself, a token of every sequence at a time; a padding row has g = beta = 0 and changes nothing."""
    q, k, v, g, beta, here, live = _padded(s, max(s.lens))
    state, o = s.pool[s.slot_in.long()], torch.empty_like(v)
    for i in range(v.shape[2]):
        state = state * torch.exp(g[:, :, i, None, None])
        u = beta[:, :, i, None] * (v[:, :, i] - (k[:, :, i, None] @ state)[:, :, 0])
        state = state + k[:, :, i, :, None] * u[:, :, None]
        o[:, :, i] = (q[:, :, i, None] @ state)[:, :, 0]
    return _packed(s, o, state, here, live)


CHUNK = 32


def _prefill_plain(s):
    """Chunks of 32 tokens: S enters a chunk; u solves the chunk's triangular system, o and the next S are products."""
    c = s.case
    n, hv, dv = c["n"], c["hv"], c["dv"]
    t = -(-max(s.lens) // CHUNK) * CHUNK
    q, k, v, g, beta, here, live = _padded(s, t)
    q, k, v = (x.reshape(n, hv, t // CHUNK, CHUNK, -1) for x in (q, k, v))
    g, beta = (x.reshape(n, hv, t // CHUNK, CHUNK) for x in (g, beta))
    cum = g.double().cumsum(-1)
    low = torch.ones(CHUNK, CHUNK, device="cuda").tril()
    decay = torch.exp((cum[..., :, None] - cum[..., None, :]).float().masked_fill(low == 0, -torch.inf))
    entry, last = torch.exp(cum.float())[..., None], torch.exp((cum[..., -1:] - cum).float())[..., None]
    system = beta[..., None] * decay * (k @ k.mT) * low.tril(-1)
    inverse = torch.eye(CHUNK, device="cuda").expand(system.shape).clone()
    for i in range(1, CHUNK):                                    # (I + system)^-1, a row at a time
        inverse[..., i, :] -= (system[..., i, None, :i] @ inverse[..., :i, :])[..., 0, :]
    inverse = inverse * beta[..., None, :]
    mix = decay * (q @ k.mT)
    state = s.pool[s.slot_in.long()]
    o = torch.empty(n, hv, t // CHUNK, CHUNK, dv, device="cuda")
    for j in range(t // CHUNK):
        u = inverse[:, :, j] @ (v[:, :, j] - entry[:, :, j] * (k[:, :, j] @ state))
        o[:, :, j] = mix[:, :, j] @ u + entry[:, :, j] * (q[:, :, j] @ state)
        state = entry[:, :, j, -1:] * state + (k[:, :, j] * last[:, :, j]).mT @ u
    return _packed(s, o.reshape(n, hv, t, dv), state, here, live)


# ---------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        x = s.x.double().reshape(-1, case["d"])
        scale = torch.full_like(x[:, :1], s.scale)
        if s.post_w is not None:
            scale = scale / (x.square().mean(1, keepdim=True) + EPS).sqrt()
            x = x * s.post_w.double()
        x = x * scale
        if s.gate is not None:
            g = s.gate.double()
            g = {"none": lambda: g, "silu": lambda: g / (1 + torch.exp(-g)), "sigmoid": lambda: 1 / (1 + torch.exp(-g))}[case["act"]]()
            x = (x.view(case["rows"], -1) * g).reshape(x.shape)
        if s.h_in is not None:
            x = x + s.h_in.double().reshape(x.shape)
        out = [x.view(case["rows"], -1)]
        if s.pre_w is not None:
            out.append((x / (x.square().mean(1, keepdim=True) + EPS).sqrt() * s.pre_w.double()).view(case["rows"], -1))
        return out
    # token by token, as the rule is defined
    n, hv, group = case["n"], case["hv"], case["hv"] // case["hk"]
    lens = torch.tensor(s.lens, device="cuda")
    start = s.seq_start[:-1].long()
    state = s.pool[s.slot_in.long()].double()
    o = torch.zeros(s.o.shape, dtype=torch.float64, device="cuda")
    every = not case["ragged"]
    for i in range(max(s.lens)):
        on = slice(None) if every else (lens > i).nonzero()[:, 0]
        row = start[on] + i
        k, q = s.k[row].double(), s.q[row].double()
        k = (k / (k.square().sum(-1, keepdim=True) + EPS).sqrt()).repeat_interleave(group, 1)
        q = (q / (q.square().sum(-1, keepdim=True) + EPS).sqrt()).repeat_interleave(group, 1) * s.scale
        S = state[on] * torch.exp(s.g[row].double())[..., None, None]
        u = s.beta[row].double()[..., None] * (s.v[row].double() - torch.einsum("nhk,nhkv->nhv", k, S))
        S = S + k[..., None] * u[..., None, :]
        o[row] = torch.einsum("nhk,nhkv->nhv", q, S)
        state[on] = S
    after = torch.empty_like(state)
    after[s.slot_out.long() - n] = state
    return o, after
