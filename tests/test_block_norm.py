"""shvk_block_norm (norm, gate, scale, residual and norm between two blocks) against its formula in float64, and what it refuses.

Tolerances.  Every step is float32.  A sum of squares is at most 64 terms a thread and a tree of ten levels (rows that no vector load
fits: 64 terms and a sum of 5 and 8), so it is off by 74 steps of 2^-24 of itself and its root by half of that; root, reciprocal,
exponential, quotient and the products add less than 60 half steps (exp's argument is rounded: |g| <= 8 here).  So y and h are within
C = 128 half steps, 128 x 2^-24, of the magnitudes that enter them, m = |h_in| + |scale y|; xn carries the error of h, that of its own
sum (C |m| / |h| as norms, relative) and C of its own.  An output's rounding adds half a step of its type.
"""
import ctypes as C

import pytest

from shield_sisa_b200 import binding

CODES = {"fp32": 0, "bf16": 1, "fp16": 2}
INVALID = 1
ERR = 128 * 2.0 ** -24


@pytest.fixture(scope="module")
def L():
    from shield_sisa_b200 import build
    build.build()
    return binding.load_library(True)


def good(**kw):
    p = 0x100000                                                # never dereferenced: every call below ends on the host
    a = dict(rows=4, heads=1, D=384, x=p, ldx=384, x_dtype=1, post_w=p, gate=p, ldgate=384, gate_dtype=1, gate_act=1, scale=1.0, h_in=p,
             ldh_in=384, h_out=p, ldh_out=384, h_dtype=0, pre_w=p, xn=p, ldxn=384, xn_dtype=1, eps=1e-6)
    a.update(kw)
    return binding.BlockNormArgs(**a)


BAD = [dict(rows=-1), dict(rows=1 << 30), dict(rows=1 << 28, heads=6, ldx=4096, ldh_in=4096, ldh_out=4096, ldxn=4096, ldgate=4096), dict(heads=0), dict(heads=5000), dict(D=0), dict(D=16385), dict(x=None), dict(x_dtype=3), dict(x_dtype=-1),
       dict(h_dtype=2), dict(h_dtype=3), dict(gate_dtype=0), dict(gate_dtype=2), dict(xn_dtype=0), dict(gate_act=3), dict(gate_act=-1),
       dict(pre_w=None), dict(xn=None), dict(pre_w=None, xn=None, h_out=None), dict(ldx=-1), dict(ldh_in=-8), dict(ldgate=-1),
       dict(ldh_out=383), dict(ldxn=376), dict(heads=2), dict(x=0x100001), dict(h_in=0x100002), dict(post_w=0x100002)]


@pytest.mark.parametrize("kw", BAD, ids=lambda d: "-".join(f"{k}={v}" for k, v in d.items()))
def test_refuses(L, kw):
    assert L.shvk_block_norm(C.byref(good(**kw)), None) == INVALID


def test_no_rows_launch_nothing(L):
    assert L.shvk_block_norm(None, None) == INVALID
    assert L.shvk_block_norm(C.byref(good(rows=0)), None) == 0


gpu = pytest.mark.gpu


def types(kind):
    import torch
    return {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}[kind]


def make(kind, rows, heads, d, post=True, gate="rows", act=1, res="fp32", pre=True, pad=0, shift=0, seed=1, h_out=True, scale=0.7):
    """A call's buffers.  pad: values between two rows; shift: values in front of the first row."""
    import torch
    gen = torch.Generator(device="cuda").manual_seed(seed)
    w = heads * d

    def rows_of(n, t, fill=None):
        flat = torch.full((shift + n * (w + pad) + 16,), 5.0, device="cuda").to(t)
        view = flat[shift:shift + n * (w + pad)].view(n, w + pad)
        view[:, :w] = torch.randn(n, w, device="cuda", generator=gen).to(t) if fill is None else fill
        return flat, view
    t, th = types(kind), types(kind if res == "none" else res)
    x = {"kind": kind, "rows": rows, "heads": heads, "d": d, "act": act, "res": res, "scale": scale, "w": w, "pad": pad, "gate_kind": gate}
    x["x_flat"], x["x"] = rows_of(rows, t)
    x["gate"] = None if gate == "none" else rows_of(rows if gate == "rows" else 1, t)[1]
    x["h_in"] = None if res == "none" else rows_of(rows, th)[1]
    x["h_flat"], x["h_out"] = rows_of(rows, th, 5.0) if h_out else (None, None)
    x["post_w"] = 1 + 0.3 * torch.randn(d, device="cuda", generator=gen) if post else None
    x["pre_w"] = 1 + 0.3 * torch.randn(d, device="cuda", generator=gen) if pre else None
    x["n_flat"], x["xn"] = rows_of(rows, t, 5.0) if pre else (None, None)
    return x


def args(x):
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    ld = lambda t: 0 if t is None else t.stride(0)  # noqa: E731
    h = x["kind"] if x["res"] == "none" else x["res"]
    return binding.BlockNormArgs(rows=x["rows"], heads=x["heads"], D=x["d"], x=ptr(x["x"]), ldx=ld(x["x"]), x_dtype=CODES[x["kind"]],
                                 post_w=ptr(x["post_w"]), gate=ptr(x["gate"]), ldgate=ld(x["gate"]) if x["gate_kind"] == "rows" else 0,
                                 gate_dtype=CODES[x["kind"]], gate_act=x["act"], scale=x["scale"], h_in=ptr(x["h_in"]),
                                 ldh_in=ld(x["h_in"]), h_out=ptr(x["h_out"]), ldh_out=ld(x["h_out"]), h_dtype=CODES[h],
                                 pre_w=ptr(x["pre_w"]), xn=ptr(x["xn"]), ldxn=ld(x["xn"]), xn_dtype=CODES[x["kind"]], eps=1e-6)


def launch(L, x, stream=None):
    import torch
    s = torch.cuda.current_stream() if stream is None else stream
    rc = L.shvk_block_norm(C.byref(args(x)), s.cuda_stream)
    assert rc == 0, rc


def formula(x):
    """(h, its tolerance, xn, its tolerance), each [rows, heads, d], without the outputs' own rounding."""
    import torch
    shape = (x["rows"], x["heads"], x["d"])
    y = x["x"][:, :x["w"]].double().reshape(shape)
    if x["post_w"] is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + 1e-6) * x["post_w"].double()
    if x["gate"] is not None:
        g = x["gate"][:, :x["w"]].double().reshape(-1, x["heads"], x["d"])
        y = y * (g if x["act"] == 0 else torch.sigmoid(g) * (g if x["act"] == 1 else 1))
    y = y * float(torch.tensor(x["scale"], dtype=torch.float32))
    h = y if x["h_in"] is None else y + x["h_in"][:, :x["w"]].double().reshape(shape)
    m = y.abs() + (h - y).abs()
    if x["pre_w"] is None:
        return h, ERR * m, None, None
    r = 1 / torch.sqrt((h * h).mean(-1, keepdim=True) + 1e-6)
    rel = m.norm(dim=-1, keepdim=True) / h.norm(dim=-1, keepdim=True).clamp_min(1e-300)
    w = x["pre_w"].double()
    return h, ERR * m, h * r * w, ERR * r * w.abs() * (m + h.abs() * (1 + rel.clamp_max(1e6)))


def check(L, x, h_in_place=False):
    import torch
    h, th, n, tn = formula(x)
    x_before = x["x_flat"].clone()
    if h_in_place:
        x["h_out"] = x["h_in"]
        x["h_flat"] = None
    launch(L, x)
    torch.cuda.synchronize()
    for out, flat, want, tol in ((x["h_out"], x["h_flat"], h, th), (x["xn"], x["n_flat"], n, tn)):
        if out is None:
            continue
        got = out[:, :x["w"]].double().reshape(want.shape)
        half = torch.finfo(out.dtype).eps / 2 if out.dtype != torch.float32 else 0.0
        tiny = 2.0 ** -25 if out.dtype == torch.float16 else 0.0
        off = (got - want).abs() - half * want.abs() - tol - tiny
        assert float(off.max()) <= 0, float(off.max())
        if flat is not None:                                    # nothing between, before or behind the rows is written
            keep = torch.ones_like(flat, dtype=torch.bool)
            start = (out.data_ptr() - flat.data_ptr()) // flat.element_size()
            keep[start:start + out.shape[0] * out.stride(0)].view(out.shape[0], out.stride(0))[:, :x["w"]] = False
            assert torch.equal(flat[keep], torch.full_like(flat[keep], 5.0))
    assert torch.equal(x["x_flat"], x_before)


WIDTHS = [1, 7, 8, 33, 120, 128, 129, 255, 256, 384, 505, 512, 513, 960, 1920, 2047, 2050, 4099, 8184, 8192, 12001, 16377, 16384]


@gpu
@pytest.mark.parametrize("kind,res", [("bf16", "fp32"), ("fp32", "fp32"), ("fp16", "fp16")])
@pytest.mark.parametrize("d", [1536, 1537, 2040, 2048, 3585, 3841, 4088, 4089, 4095, 4096, 4097, 8177, 8191, 8193])
def test_widths_where_the_shared_memory_changes(L, kind, res, d):
    """Weights and rows of a CTA around the sizes at which a launch has to ask for more than 48 KB, with and without all of them."""
    check(L, make(kind, 9, 1, d, res=res, seed=d + 1))
    check(L, make(kind, 9, 1, d, res=res, seed=d + 2, gate="one"))


@gpu
@pytest.mark.parametrize("kind,res", [("bf16", "fp32"), ("fp16", "fp16"), ("fp32", "fp32"), ("bf16", "bf16"), ("fp16", "fp32")])
@pytest.mark.parametrize("d", WIDTHS)
def test_every_width(L, kind, res, d):
    check(L, make(kind, 21, 1, d, res=res, seed=d))


@gpu
@pytest.mark.parametrize("d", [33, 384, 2047, 4099])
@pytest.mark.parametrize("rows", [1, 2, 9, 1203])
def test_rows_of_a_long_call(L, d, rows):
    check(L, make("bf16", rows, 1, d, gate="one", act=2, seed=rows))


@gpu
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("gate,act", [("none", 0), ("rows", 0), ("rows", 1), ("rows", 2), ("one", 0), ("one", 1)])
@pytest.mark.parametrize("res,pre,h_out", [("none", False, True), ("none", True, True), ("fp32", True, True), ("fp32", False, True), ("bf16", True, False)])
def test_every_part_left_out(L, post, gate, act, res, pre, h_out):
    for d in (384, 61, 2047):
        check(L, make("bf16", 13, 1, d, post=post, gate=gate, act=act, res=res, pre=pre, h_out=h_out, seed=d))


@gpu
@pytest.mark.parametrize("d", [128, 64, 20, 27])
@pytest.mark.parametrize("gate", ["none", "rows", "one"])
def test_heads_of_a_row(L, d, gate):
    for rows in (1, 3, 500):
        check(L, make("bf16", rows, 6, d, gate=gate, res="none", pre=False, seed=rows))
        check(L, make("fp16", rows, 6, d, gate=gate, res="fp32", pad=24, seed=rows))


@gpu
@pytest.mark.parametrize("d,pad,shift", [(384, 8, 0), (384, 1, 0), (384, 0, 1), (384, 4, 8), (100, 2, 0), (100, 0, 0), (255, 1, 0), (255, 3, 5),
                                         (2047, 2, 16), (1022, 0, 0), (1020, 0, 3)])
def test_pitches_and_starts(L, d, pad, shift):
    for kind, res in (("bf16", "fp32"), ("fp32", "fp32")):
        check(L, make(kind, 19, 1, d, res=res, pad=pad, shift=shift, seed=d + pad))


@gpu
def test_arrays_that_start_at_different_places(L):
    """No vector load fits all arrays of the call."""
    x = make("bf16", 11, 1, 384, seed=3)
    y = make("bf16", 11, 1, 384, pad=3, seed=4)
    x["gate"], x["h_in"] = y["gate"], y["h_in"]
    check(L, x)


@gpu
@pytest.mark.parametrize("d", [384, 61, 2047, 16384])
def test_residual_in_place(L, d):
    check(L, make("bf16", 23, 1, d, res="fp32", seed=d), h_in_place=True)
    check(L, make("fp16", 23, 1, d, res="fp16", seed=d, pad=1), h_in_place=True)


@gpu
@pytest.mark.parametrize("d", [384, 61, 2047])
def test_output_over_the_input(L, d):
    import torch
    x = make("bf16", 37, 1, d, res="none", pre=False, seed=d)
    want = formula(x)[0]
    x["h_out"] = x["x"]
    launch(L, x)
    torch.cuda.synchronize()
    got = x["x"][:, :d].double().view(want.shape)
    assert float(((got - want).abs() - (2.0 ** -8 + 2 * ERR) * want.abs()).max()) <= 0


@gpu
@pytest.mark.parametrize("d", [128, 384, 2047, 15999])
def test_zeros_infinities_and_nan_stay_in_their_row(L, d):
    import torch
    x, y = make("bf16", 17, 1, d, seed=1), make("bf16", 17, 1, d, seed=1)
    x["x"][3, :d] = 0
    x["h_in"][3, :d] = 0
    x["x"][5, d // 2] = float("nan")
    x["x"][9, 0] = float("inf")
    x["h_in"][11, d - 1] = -float("inf")
    launch(L, x)
    launch(L, y)
    torch.cuda.synchronize()
    for name in ("h_out", "xn"):
        assert not x[name][3, :d].any()                         # 0 / sqrt(0 + eps)
        assert torch.isnan(x[name][5, :d].float()).any()
        for r in range(17):
            if r not in (3, 5, 9, 11):
                assert torch.equal(x[name][r], y[name][r])


@gpu
def test_a_row_gives_the_same_bits_alone(L):
    import torch
    for d in (384, 2047):
        x = make("bf16", 1500, 1, d, seed=7)
        launch(L, x)
        for r in (0, 8, 777, 1499):                             # rows that start on a group of eight when they are alone as well
            if (r * d) % 8:
                continue
            y = dict(x)
            y["rows"] = 1
            for name in ("x", "gate", "h_in"):
                y[name] = x[name][r:r + 1]
            y["h_out"], y["xn"] = torch.empty_like(x["h_out"][:1]), torch.empty_like(x["xn"][:1])
            launch(L, y)
            torch.cuda.synchronize()
            assert torch.equal(y["h_out"][0], x["h_out"][r]) and torch.equal(y["xn"][0], x["xn"][r])


@gpu
def test_captured_and_replayed(L):
    import torch
    x, y = make("bf16", 40, 1, 384, seed=1), make("bf16", 40, 1, 384, seed=2)
    launch(L, x)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        launch(L, x)
    for name in ("x", "gate", "h_in", "post_w", "pre_w"):
        x[name].copy_(y[name])
    graph.replay()
    launch(L, y)
    torch.cuda.synchronize()
    assert torch.equal(x["h_out"], y["h_out"]) and torch.equal(x["xn"], y["xn"])


@gpu
@pytest.mark.parametrize("d", [128, 384, 2047, 2048, 16377])
def test_norms_behind_one_another(L, d):
    """Each call reads what the one before wrote, in place and with nothing between them: the same bits as with a pause behind each."""
    import torch
    x = make("bf16", 700, 1, d, res="fp32", gate="none", seed=3 + d)
    y = dict(x)
    y["x"], y["xn"] = x["xn"], x["x"]                            # the other way round, h in place
    x["h_out"] = y["h_out"] = y["h_in"] = x["h_in"]
    first = [x[name].clone() for name in ("x", "xn", "h_in")]

    def run(pause):
        for name, v in zip(("x", "xn", "h_in"), first):
            x[name].copy_(v)
        for i in range(12):
            launch(L, (x, y)[i % 2])
            if pause:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        return [x[name].clone() for name in ("x", "xn", "h_in")]
    want = run(True)
    assert all(torch.isfinite(w.float()).all() for w in want)
    for _ in range(5):
        assert all(torch.equal(g, w) for g, w in zip(run(False), want))


GROUPS = r"""
#include <cuda_runtime.h>
#include "block_norm_rows.cuh"
#include <cstdio>
// every group that a row of the kernel takes, for rows, pitch and width: reads outside the array, whole groups over a row's end
int main() {
    long long outside = 0, over = 0, groups = 0;
    for (int D = 1; D <= 40; ++D)
        for (long long ld = 0; ld <= 3 * D + 17; ++ld)
            for (int rows = 1; rows <= 40; ++rows) {
                const int P = ld % 8 == 0 ? 1 : ld % 2 ? 8 : ld % 4 ? 4 : 2, whole = sb::whole_rows(rows, ld);
                const long long size = (rows - 1) * ld + D;
                for (int row = 0; row < rows; ++row) {
                    const int off = sb::row_shift(row % P, ld);
                    if ((row * ld - off) % 8) return 1;          // a group starts where the loads do
                    int seen = 0;
                    for (int c = -off; c < D; c += 8) {
                        const int lo = sb::group_lo(c), hi = sb::group_hi(c, D);
                        if (hi <= lo) continue;
                        const bool all = sb::reads_whole(c + 8, D, row, whole);
                        const long long first = row * ld + c + (all ? 0 : lo), last = row * ld + c + (all ? 8 : hi);
                        outside += first < 0 || last > size;
                        over += all && hi < 8;
                        seen += hi - lo;
                        ++groups;
                    }
                    if (seen != D) return 2;
                }
            }
    printf("%lld %lld %lld\n", groups, outside, over);
}
"""


def test_no_group_is_read_past_its_array(tmp_path):
    """The kernel's own rules for groups of eight, compiled for the host, over all small widths, pitches and numbers of rows."""
    import subprocess

    from shield_sisa_b200 import build
    src, exe = tmp_path / "groups.cu", tmp_path / "groups"
    src.write_text(GROUPS)
    subprocess.run([build.NVCC, *build.NVCC_FLAGS, str(src), "-o", str(exe)], check=True, capture_output=True)
    groups, outside, over = (int(v) for v in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split())
    assert outside == 0 and groups > 1 << 20 and over > 1 << 18


@gpu
@pytest.mark.parametrize("kind,res", [("bf16", "fp32"), ("fp32", "fp32"), ("fp16", "fp16")])
@pytest.mark.parametrize("d", [1, 2, 3, 4, 5, 6, 7, 9, 11, 13])
def test_small_widths_in_arrays_without_a_tail(L, kind, res, d):
    import torch
    for rows in (1, 2, 3, 6, 9, 25):
        x = make(kind, rows, 1, d, res=res, seed=d)
        for name in ("x", "gate", "h_in", "h_out", "xn"):
            x[name] = x[name].clone()
        x["h_flat"] = x["n_flat"] = None
        assert x["x"].untyped_storage().nbytes() == rows * d * x["x"].element_size()
        check(L, x)


@gpu
def test_calls_of_two_threads_do_not_take_each_others_shared_memory(L):
    """Widths that ask for little and for much shared memory, launched by two host threads at once: no call may refuse or change for the
    other's sake.  (The limit of a kernel is one for all of its callers.)"""
    import threading

    import torch
    wide = [make("bf16", 2, 1, 16384, res="fp32", seed=1, pad=8), make("bf16", 2, 1, 16380, res="fp32", seed=2, shift=1),
            make("bf16", 2, 1, 6000, res="fp32", seed=3), make("bf16", 2, 1, 4095, res="fp32", seed=3)]
    small = [make("bf16", 2, 1, 8200, res="fp32", seed=4, pad=8), make("bf16", 2, 1, 100, res="fp32", seed=5, shift=1),
             make("bf16", 2, 1, 4160, res="fp32", seed=6), make("bf16", 2, 1, 521, res="fp32", seed=3)]
    torch.cuda.synchronize()
    streams, codes = [torch.cuda.Stream(), torch.cuda.Stream()], [set(), set()]

    def work(i, calls):
        torch.cuda.set_device(0)
        packed = [args(x) for x in calls]
        for _ in range(3000):
            for a in packed:
                codes[i].add(L.shvk_block_norm(C.byref(a), streams[i].cuda_stream))
    threads = [threading.Thread(target=work, args=(i, calls)) for i, calls in enumerate((wide, small))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert codes == [{0}, {0}], codes
    for x in wide + small:
        check(L, x)


@gpu
def test_a_small_call_behind_a_large_one_in_a_graph(L):
    """Both captured before the graph is made."""
    import torch
    calls = [make("bf16", 3, 1, d, res="fp32", seed=d, shift=s) for d, s in ((16384, 1), (100, 1), (8200, 0), (4160, 0))]
    for x in calls:
        launch(L, x)
    torch.cuda.synchronize()
    want = [(x["h_out"].clone(), x["xn"].clone()) for x in calls]
    for order in (calls, calls[::-1]):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for x in order:
                launch(L, x)
        for x in calls:
            x["h_out"].zero_(), x["xn"].zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x["h_out"], w[0]) and torch.equal(x["xn"], w[1]) for x, w in zip(calls, want))


@gpu
@pytest.mark.parametrize("kind,res,h", [("bf16", "none", "fp32"), ("fp16", "none", "fp32"), ("bf16", "fp32", "fp32"), ("fp32", "none", "fp32"),
                                        ("bf16", "none", "bf16"), ("fp16", "fp16", "fp16")])
@pytest.mark.parametrize("act", [1, 2])
@pytest.mark.parametrize("d", [384, 61, 2048, 12001])
@pytest.mark.parametrize("gate", ["rows", "one"])
def test_gates_far_from_zero(L, kind, res, h, act, d, gate):
    """Gates of -100 to 100: float32 outputs are float32's although the gate has 16 bits, and a gate that is nearly closed is not taken for
    a closed one (x of up to 2^100 behind it: values far above a type's smallest).  exp and the quotient stay within the half steps that
    stand above; where exp's own result is subnormal it is off by 2^-149.  16-bit outputs come from a shorter exponential, whose argument
    of up to 145 is rounded to 24 bits: 145 x 2^-24 and 2^-22, 2^-16 of the value in all, on top of their own rounding."""
    import torch
    x = make(kind, 9, 1, d, post=False, gate=gate, act=act, res=res, pre=False, seed=d, scale=1.0)
    t, th = types(kind), types(h)
    x["gate"][:, :d] = (200 * torch.rand(x["gate"].shape[0], d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(d)) - 100).to(t)
    if kind != "fp16":
        x["x"][::2, :d] = (x["x"][::2, :d].float() * 2.0 ** 100).to(t)
    if res == "none":
        x["h_flat"], x["h_out"] = None, torch.full((9, d), 5.0, device="cuda", dtype=th)
    a = args(x)
    a.h_dtype = CODES[h]
    assert L.shvk_block_norm(C.byref(a), torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    y, g = x["x"][:, :d].double(), x["gate"][:, :d].double()
    want = y * torch.sigmoid(g) * (g if act == 1 else 1)
    off = (ERR + (0.0 if h == "fp32" else 2.0 ** -16)) * want.abs() + (y * (g if act == 1 else 1)).abs() * 2.0 ** -148
    if res != "none":
        r = x["h_in"][:, :d].double()
        want, off = want + r, off + ERR * r.abs()
    got = x["h_out"][:, :d].double()
    half = torch.finfo(th).eps / 2
    tiny = 2.0 ** -25 if h == "fp16" else 2.0 ** -149 if h == "fp32" else 2.0 ** -134
    assert float(((got - want).abs() - half * want.abs() - off - tiny).max()) <= 0


@gpu
@pytest.mark.parametrize("d", [5, 128, 384, 2047, 2048, 12001])
def test_the_next_norm_over_the_input(L, d):
    """xn over x and h over the residual, at once: the same bits as into arrays of their own."""
    import torch
    x, y = make("bf16", 301, 1, d, seed=d), make("bf16", 301, 1, d, seed=d)
    launch(L, x)
    y["xn"], y["h_out"] = y["x"], y["h_in"]
    launch(L, y)
    torch.cuda.synchronize()
    assert torch.equal(x["xn"], y["x"]) and torch.equal(x["h_out"], y["h_in"])


@gpu
@pytest.mark.parametrize("d,pad", [(384, 0), (381, 0), (384, 3)])
def test_rows_past_two_gigabytes(L, d, pad):
    """More than 2^31 values in an array: the last rows as they come out alone."""
    import torch
    rows = (1 << 31) // (d + pad) + 100
    rows += -rows % 8                                            # (the last eight rows start at the places that eight rows alone have)
    gen = torch.Generator(device="cuda").manual_seed(d)
    flat = torch.zeros(rows * (d + pad) + 16, device="cuda", dtype=torch.bfloat16)
    shift = 1 if pad else 0
    big = flat[shift:shift + rows * (d + pad)].view(rows, d + pad)
    last = torch.randn(8, d, device="cuda", generator=gen).bfloat16()
    big[-8:, :d] = last
    w = 1 + 0.3 * torch.randn(d, device="cuda", generator=gen)

    def norm(x, n):
        a = binding.BlockNormArgs(rows=n, heads=1, D=d, x=x.data_ptr(), ldx=d + pad, x_dtype=1, post_w=w.data_ptr(), scale=0.5, h_out=x.data_ptr(),
                                  ldh_out=d + pad, h_dtype=1, eps=1e-6)
        assert L.shvk_block_norm(C.byref(a), torch.cuda.current_stream().cuda_stream) == 0
    small_flat = torch.zeros(8 * (d + pad) + 16, device="cuda", dtype=torch.bfloat16)
    small = small_flat[shift:shift + 8 * (d + pad)].view(8, d + pad)
    small[:, :d] = last
    norm(big, rows)
    norm(small, 8)
    torch.cuda.synchronize()
    assert torch.equal(big[-8:], small) and not flat[:(rows - 8) * (d + pad)].any()
    assert torch.isfinite(small.float()).all() and small[:, :d].any(dim=1).all()
    del big, flat
    torch.cuda.empty_cache()
