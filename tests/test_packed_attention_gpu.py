"""Causal attention over packed prompts with grouped heads
(fml_attention_packed) against the formula in 64 bits.

The tolerance of an output element is A * (relative error of its
probabilities) + |o| u, with A = sum_j p_j |v_j|: a score is off by at most
scale sum |q||k| (hd + 4) 2^-23 (products and their sum in 32 bits, or three
TF32 products), the exponent's argument and 2^x by 2^-20 + |s| 2^-23, a sum of n
terms by n 2^-24, each twice (numerator and denominator); 16-bit inputs round
p once (u = 2^-11, 2^-8) and the result once."""
import math

import numpy as np
import pytest
import torch

from freeml_b200 import _lib, matrix_ops

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
U = {"fp32": 0.0, "fp16": 2.0 ** -11, "bf16": 2.0 ** -8}


def starts_of(lens):
    return torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")


def make(lq, lk, heads, kv, hd, kind, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randn(sum(lq), heads, hd, generator=g, device="cuda").to(DT[kind])
    k = torch.randn(sum(lk), kv, hd, generator=g, device="cuda").to(DT[kind])
    v = torch.randn(sum(lk), kv, hd, generator=g, device="cuda").to(DT[kind])
    return q, k, v


def reference(q, k, v, lq, lk, scale, kind, lossy=0.0):
    """(output, tolerance) in 64 bits."""
    group, hd = q.shape[1] // k.shape[1], q.shape[2]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    qa = ka = 0
    for nq, nk in zip(lq, lk):
        if nq:
            seen = torch.arange(nk, device="cuda")[None] <= torch.arange(nq, device="cuda")[:, None] + (nk - nq)
            any_ = seen.any(1)
            for h in range(q.shape[1]):
                Q, K, V = q[qa:qa + nq, h].double(), k[ka:ka + nk, h // group].double(), v[ka:ka + nk, h // group].double()
                s = (Q @ K.T * scale).masked_fill(~seen, -math.inf)
                ds = (Q.abs() @ K.abs().T * scale * ((hd + 4) * 2.0 ** -23 + lossy)).masked_fill(~seen, 0.0)
                big = s.masked_fill(~seen, 0.0).abs()
                p = torch.zeros_like(s)
                p[any_] = torch.softmax(s[any_], -1)
                o = p @ V
                A = p @ V.abs()
                rel = 2 * (ds + big * 2.0 ** -23).amax(-1, keepdim=True) if nk else torch.zeros(nq, 1, device="cuda")
                rel = rel + 2.0 ** -19 + nk * 2.0 ** -23 + U[kind] + lossy
                out[qa:qa + nq, h] = o
                tol[qa:qa + nq, h] = A * rel + o.abs() * U[kind]
        qa, ka = qa + nq, ka + nk
    return out, tol


def check(got, want, tol):
    assert torch.isfinite(got).all()
    worst = ((got.double() - want).abs() - tol).max().item() if got.numel() else 0.0
    assert worst <= 0.0, worst


LENS = {
    "one": [1],
    "tiny": [3, 1, 0, 2],
    "edges": [63, 64, 65, 127, 128, 129, 1],
    "wide": [255, 256, 257, 0, 300, 17],
    "long": [1000, 7],
}


@pytest.mark.parametrize("lens", sorted(LENS))
@pytest.mark.parametrize("heads,kv,hd", [(4, 4, 32), (6, 2, 64), (8, 8, 64), (8, 1, 128), (10, 2, 128), (3, 3, 128)])
@pytest.mark.parametrize("kind", sorted(DT))
def test_prompts(kind, heads, kv, hd, lens):
    lq = LENS[lens]
    q, k, v = make(lq, lq, heads, kv, hd, kind)
    out = torch.full_like(q, float("nan"))
    scale = 1.0 / math.sqrt(hd)
    matrix_ops.attention_packed(out, q, k, v, starts_of(lq), scale)
    check(out, *reference(q, k, v, lq, lq, scale, kind))


@pytest.mark.parametrize("kind", sorted(DT))
@pytest.mark.parametrize("heads,kv,hd", [(4, 4, 32), (2, 1, 64), (4, 1, 128)])
@pytest.mark.parametrize("n", [1280, 1537, 2300, 4095])
def test_many_key_tiles(kind, heads, kv, hd, n):
    """Every stage of the copies' ring is used more than once, and the last key
    tile is whole, or ends inside the sequence's last rows."""
    lq, lk = [n, 60, 130], [n, n + 60, n + 130]
    q, k, v = make(lq, lk, heads, kv, hd, kind, 9)
    v[n + n + 60:][:n] += 1.0
    out = torch.full_like(q, float("nan"))
    scale = 1.0 / math.sqrt(hd)
    matrix_ops.attention_packed(out, q, k, v, starts_of(lq), scale, k_starts=starts_of(lk))
    check(out, *reference(q, k, v, lq, lk, scale, kind))


@pytest.mark.parametrize("kind", sorted(DT))
@pytest.mark.parametrize("heads,kv,hd", [(4, 4, 64), (8, 2, 128), (4, 1, 32)])
def test_keys_lead_or_lag_the_queries(kind, heads, kv, hd):
    """Chunks after a prefix; and sequences with fewer keys than rows, whose
    first rows see none and are zero."""
    lq = [5, 130, 1, 64, 40, 7, 200]
    lk = [205, 131, 77, 64, 13, 0, 390]
    q, k, v = make(lq, lk, heads, kv, hd, kind, 1)
    out = torch.full_like(q, float("nan"))
    scale = 0.3
    matrix_ops.attention_packed(out, q, k, v, starts_of(lq), scale, k_starts=starts_of(lk))
    want, tol = reference(q, k, v, lq, lk, scale, kind)
    check(out, want, tol)
    at = sum(lq[:4])
    assert (out[at:at + 27] == 0).all() and (out[at + 40:at + 47] == 0).all()


@pytest.mark.parametrize("kind", sorted(DT))
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_wide_groups(kind, hd):
    """More query heads to a key/value head than a tile has rows for a token."""
    lq = [9, 33]
    q, k, v = make(lq, lq, 140, 1, hd, kind, 2)
    out = torch.full_like(q, float("nan"))
    matrix_ops.attention_packed(out, q, k, v, starts_of(lq), 0.1)
    check(out, *reference(q, k, v, lq, lq, 0.1, kind))


@pytest.mark.parametrize("kind", sorted(DT))
@pytest.mark.parametrize("shift", [0, 1])
def test_views_of_one_row_and_odd_bases(kind, shift):
    """q, k and v as views of one QKV row; an output with its own stride; and
    bases and strides that no wide access can be used on."""
    lq, heads, kv, hd = [70, 200, 3], 6, 2, 64
    width = (heads + 2 * kv) * hd + shift
    T = sum(lq)
    flat = torch.randn(T * width + 8, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).to(DT[kind])
    rows = flat[shift:shift + T * width].view(T, width)
    q, k, v = (rows[:, a * hd:b * hd].unflatten(1, (b - a, hd)) for a, b in ((0, heads), (heads, heads + kv), (heads + kv, heads + 2 * kv)))
    whole = torch.full((T + 2, heads * hd + 16 + shift), 7.0, device="cuda", dtype=DT[kind])
    out = whole[1:-1, 8:8 + heads * hd].unflatten(1, (heads, hd))
    matrix_ops.attention_packed(out, q, k, v, starts_of(lq), 0.125)
    check(out, *reference(q, k, v, lq, lq, 0.125, kind))
    mask = torch.ones_like(whole, dtype=torch.bool)
    mask[1:-1, 8:8 + heads * hd] = False
    assert (whole[mask] == 7.0).all()


@pytest.mark.parametrize("kind", sorted(DT))
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_other_sequences_never_reach_a_row(kind, hd):
    """Neighbours full of NaN and infinities, rows of no sequence among them."""
    lq = [40, 30, 100, 25, 90]
    q, k, v = make(lq, lq, 4, 2, hd, kind, 4)
    at = np.cumsum([0] + lq)
    bad = torch.zeros(len(q), dtype=torch.bool, device="cuda")
    for i in (1, 3):
        bad[at[i]:at[i + 1]] = True
    clean = reference(q, k, v, lq, lq, 0.2, kind)
    for t in (q, k, v):
        t[bad] = float("nan")
    v[bad] = float("inf")
    out = torch.empty_like(q)
    matrix_ops.attention_packed(out, q, k, v, starts_of(lq), 0.2)
    check(out[~bad], clean[0][~bad], clean[1][~bad])


@pytest.mark.parametrize("kind", sorted(DT))
def test_rows_of_no_sequence_are_left(kind):
    q, k, v = make([100], [100], 4, 4, 64, kind, 5)
    out = torch.full_like(q, 5.0)
    starts = torch.tensor([10, 40, 90], dtype=torch.int32, device="cuda")
    matrix_ops.attention_packed(out, q, k, v, starts, 0.2)
    assert (out[:10] == 5).all() and (out[90:] == 5).all()
    want, tol = reference(q[10:90], k[10:90], v[10:90], [30, 50], [30, 50], 0.2, kind)
    check(out[10:90], want, tol)
    # starts past the rows are cut to them
    starts = torch.tensor([10, 40, 1000], dtype=torch.int32, device="cuda")
    matrix_ops.attention_packed(out, q, k, v, starts, 0.2)
    want, tol = reference(q[10:], k[10:], v[10:], [30, 60], [30, 60], 0.2, kind)
    check(out[10:], want, tol)


@pytest.mark.parametrize("kind", sorted(DT))
@pytest.mark.parametrize("hd", [64, 128])
def test_rising_and_far_scores(kind, hd):
    """Maxima that rise along the keys by far more than one tile's scores vary,
    so that earlier sums are rescaled; and scores far from zero."""
    n = 700
    g = torch.Generator(device="cuda").manual_seed(6)
    q = torch.randn(n, 2, hd, generator=g, device="cuda").to(DT[kind])
    k = (torch.randn(n, 1, hd, generator=g, device="cuda") * torch.linspace(0.1, 6.0, n, device="cuda")[:, None, None]).to(DT[kind])
    v = torch.randn(n, 1, hd, generator=g, device="cuda").to(DT[kind])
    out = torch.empty_like(q)
    matrix_ops.attention_packed(out, q, k, v, starts_of([n]), 0.5)
    check(out, *reference(q, k, v, [n], [n], 0.5, kind))


@pytest.mark.parametrize("mode,lossy", [(_lib.FML_MATH_FP32, 0.0), (_lib.FML_MATH_TF32X3, 0.0), (_lib.FML_MATH_TF32, 2.0 ** -9)])
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_fp32_modes(mode, lossy, hd):
    lq = [300, 129, 5]
    q, k, v = make(lq, lq, 8, 4, hd, "fp32", 7)
    out = torch.empty_like(q)
    matrix_ops.attention_packed(out, q, k, v, starts_of(lq), 0.15, mode=mode)
    check(out, *reference(q, k, v, lq, lq, 0.15, "fp32", lossy))


def test_many_sequences_and_a_stream_of_its_own():
    rng = np.random.RandomState(8)
    lq = [int(x) for x in rng.randint(0, 9, 1500)]
    q, k, v = make(lq, lq, 4, 2, 64, "bf16", 8)
    starts = starts_of(lq)
    out = torch.empty_like(q)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        matrix_ops.attention_packed(out, q, k, v, starts, 0.2)
    st.synchronize()
    some = [0, 1, 700, 1498, 1499]
    at = np.cumsum([0] + lq)
    for i in some:
        if lq[i]:
            a, b = at[i], at[i + 1]
            want, tol = reference(q[a:b], k[a:b], v[a:b], [lq[i]], [lq[i]], 0.2, "bf16")
            check(out[a:b], want, tol)
    again = torch.empty_like(q)
    matrix_ops.attention_packed(again, q, k, v, starts, 0.2)
    assert torch.equal(out, again)


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("kind", sorted(DT))
def test_scales_that_are_not_positive(kind, hd):
    lq = [1, 200, 0, 77]
    q, k, v = make(lq, lq, 6, 2, hd, kind, 17)
    for scale, same in ((-0.15, -q), (0.0, 0 * q)):
        out = torch.full_like(q, float("nan"))
        matrix_ops.attention_packed(out, q, k, v, starts_of(lq), scale)
        check(out, *reference(same, k, v, lq, lq, 0.15, kind))


def test_no_wait_ran_out():
    import ctypes
    n = ctypes.c_uint64(1)
    _lib.call("fml_device_error_count", ctypes.byref(n))
    assert n.value == 0


def test_refusals():
    q, k, v = make([8], [8], 4, 2, 64, "bf16")
    s = starts_of([8])
    out = torch.empty_like(q)
    with pytest.raises(_lib.FmlError):
        matrix_ops.attention_packed(out, q, k.float(), v.float(), s, 0.1)
    with pytest.raises(_lib.FmlError):
        matrix_ops.attention_packed(out, q, k[..., :32], v[..., :32], s, 0.1)
    with pytest.raises(_lib.FmlError):
        matrix_ops.attention_packed(out, q, k[:, :1].expand(-1, 3, -1), v[:, :1].expand(-1, 3, -1), s, 0.1)
    with pytest.raises(_lib.FmlError):
        matrix_ops.attention_packed(out, q, k, v, s.long(), 0.1)
    with pytest.raises(_lib.FmlError):
        matrix_ops.attention_packed(out.float(), q.float(), k.float(), v.float(), s, 0.1, mode=9)
    empty = q[:0]
    matrix_ops.attention_packed(out[:0], empty, k[:0], v[:0], starts_of([0]), 0.1)  # nothing to do


@pytest.mark.parametrize("heads,kv,hd", [(6, 2, 32), (4, 4, 64), (4, 1, 128)])
@pytest.mark.parametrize("lq,lk", [([512], [3300]), ([12] * 3, [900, 905, 910]), ([2048, 700], [2048, 700])])
def test_fp32_error_does_not_grow_with_the_keys(heads, kv, hd, lq, lk):
    """The 2-norm of the error over the result's, which the keys' number does
    not enter.  A tile's P V: 8 sums cut by 2^-24 or less, 5e-7; p: 2^x, its two
    TF32 parts and its argument, 2^-22 each, 7e-7; scores of about 1: hd / 8 cut
    sums that grow to it, 2^-24 hd / 16 on average, 5e-7 at most.  Together 2e-6."""
    q, k, v = make(lq, lk, heads, kv, hd, "fp32", 9)
    out = torch.empty_like(q)
    scale = hd ** -0.5
    matrix_ops.attention_packed(out, q, k, v, starts_of(lq), scale, k_starts=starts_of(lk))
    want, _ = reference(q, k, v, lq, lk, scale, "fp32")
    assert ((out.double() - want).norm() / want.norm()).item() <= 2e-6
