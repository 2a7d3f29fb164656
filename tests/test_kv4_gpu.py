"""The 4-bit paged key/value cache: rows written and read back, its attention
against the formula in 64 bits, and its page operations against a plain model."""
import math

import numpy as np
import pytest
import torch

from freeml_b200 import FmlError, kv4

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
U = {"fp32": 2.0 ** -24, "fp16": 2.0 ** -11, "bf16": 2.0 ** -8}


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def starts_of(lens):
    return ints(np.concatenate([[0], np.cumsum(lens)]).tolist())


def quantised(x):
    """numpy float32 [..., hd] -> the values that the format keeps, restated step by step in float32."""
    g = np.clip(x.astype(np.float32), -65504.0, 65504.0).reshape(*x.shape[:-1], -1, 32)
    with np.errstate(all="ignore"):
        mn = g.min(-1, keepdims=True).astype(np.float16).astype(np.float32)
        sc = ((g.max(-1, keepdims=True) - mn) * np.float32(1 / 15)).astype(np.float16).astype(np.float32)
        inv = np.where(sc == 0, np.float32(0), np.float32(1) / sc)
        c = np.clip(np.rint((g - mn) * inv), 0, 15)
        bad = np.isnan(g).any(-1, keepdims=True)
        y = mn + np.where(bad, 0, c) * sc
    return np.where(bad, np.nan, y).reshape(x.shape).astype(np.float32)


def rows(lens, kv, hd, kind, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    k = torch.randn(sum(lens), kv, hd, generator=g, device="cuda") + 2 * torch.randn(kv, hd, generator=g, device="cuda")
    v = torch.randn(sum(lens), kv, hd, generator=g, device="cuda") * 0.3
    return k.to(DT[kind]), v.to(DT[kind])


def cache_with(lens, kv, hd, page, kind="fp32", seed=0, slots=None, order=None):
    """A cache that holds the rows of rows(...), its free pages full of 0xff
    bytes (pairs that are NaN) and its pages handed out in no order."""
    slots = len(lens) if slots is None else slots
    need = [-(-n // page) for n in lens]
    c = kv4.KV4Cache(1, kv, hd, sum(need) + 3, page, slots, max(need + [1]) + 1)
    c.pool.fill_(255)
    perm = np.random.RandomState(seed).permutation(sum(need) + 3)
    table, at = c.table.cpu(), 0
    order = list(range(len(lens))) if order is None else order
    for s, n, w in zip(order, lens, need):
        table[s, :w] = torch.from_numpy(perm[at:at + w].astype(np.int32))
        at += w
        c.lens[s] = n
    c.table.copy_(table)
    k, v = rows(lens, kv, hd, kind, seed)
    c.append(0, k, v, starts_of(lens), ints(order))
    return c, k, v


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("kind", sorted(DT))
def test_rows_come_back_as_the_format_says(kind, hd, page):
    lens = [1, 0, 17, 64, 130, 5]
    c, k, v = cache_with(lens, 3, hd, page, kind, 1)
    ko = torch.empty(k.shape, device="cuda")
    vo = torch.empty(v.shape, device="cuda")
    c.read(0, ko, vo, starts_of(lens))
    np.testing.assert_array_equal(ko.cpu().numpy(), quantised(k.float().cpu().numpy()))
    np.testing.assert_array_equal(vo.cpu().numpy(), quantised(v.float().cpu().numpy()))
    # in the inputs' type: the same values rounded once
    kt, vt = torch.empty_like(k), torch.empty_like(v)
    c.read(0, kt, vt, starts_of(lens))
    assert torch.equal(kt, ko.to(k.dtype)) and torch.equal(vt, vo.to(v.dtype))


@pytest.mark.parametrize("hd", [32, 64, 128])
def test_bytes_are_the_documented_layout(hd):
    """Every column's code and pair, found by the header's words."""
    page, kv, n = 32, 2, 40
    c, k, v = cache_with([n], kv, hd, page, "fp32", 2)
    table, raw = c.table[0].tolist(), c.pool[0].cpu().numpy().reshape(c.pool.shape[1], kv, -1)
    NG, half = hd // 32, page * hd // 2 + page * hd // 8
    want = [quantised(x.cpu().numpy()) for x in (k, v)]
    for t in (0, 15, 31, 32, 39):
        for h in range(kv):
            block = raw[table[t // page], h]
            for which, unit in ((0, 8), (1, 4)):
                part = block[which * half:(which + 1) * half]
                codes = part[(t % page) * (hd // 2):][:hd // 2]
                pairs = part[page * hd // 2:].view(np.float16).reshape(page, NG, 2)[t % page].astype(np.float32)
                for d in range(hd):
                    g, u, i = d // 32, d % 32 // unit, d % unit
                    nib = (u * NG + g) * unit + i
                    code = (int(codes[nib // 2]) >> (4 * (nib % 2))) & 15
                    assert pairs[g, 1] + np.float32(code) * pairs[g, 0] == want[which][t, h, d]


def test_groups_that_are_odd():
    """Constant groups, extremes past fp16, infinities, NaN, tiny ranges."""
    hd, page = 64, 16
    x = torch.randn(8, 1, hd, device="cuda")
    x[0] = 3.25
    x[1, 0, :32] = 0.0
    x[2, 0, 5] = 1e30
    x[3, 0, 40] = float("-inf")
    x[3, 0, 3] = float("inf")
    x[4, 0, 33] = float("nan")
    x[5] *= 1e-7
    x[6] = 1000 + 1e-3 * x[6]
    x[7, 0, 0], x[7, 0, 31] = -65504.0, 65504.0
    c = kv4.KV4Cache(1, 1, hd, 2, page, 1, 2)
    c.reserve(ints([8]))
    c.append(0, x, x, starts_of([8]))
    ko, vo = torch.empty_like(x), torch.empty_like(x)
    c.read(0, ko, vo, starts_of([8]))
    want = quantised(x.cpu().numpy())
    np.testing.assert_array_equal(ko.cpu().numpy(), want)
    np.testing.assert_array_equal(vo.cpu().numpy(), want)
    assert np.isnan(want[4, 0, 32:]).all() and np.isfinite(want[4, 0, :32]).all()


@pytest.mark.parametrize("kind", sorted(DT))
@pytest.mark.parametrize("shift", [0, 1])
def test_strided_rows_and_rows_without_a_place(kind, shift):
    """Views of one QKV row, odd bases; a sequence shorter than its new rows,
    a slot and a page that do not exist: those rows are passed over."""
    hd, kv, page = 64, 2, 16
    lens = [20, 6, 9]
    T, width = sum(lens), 6 * hd + shift
    flat = torch.randn(T * width + 4, device="cuda").to(DT[kind])
    both = flat[shift:shift + T * width].view(T, width)
    k, v = both[:, hd:3 * hd].unflatten(1, (kv, hd)), both[:, 3 * hd:5 * hd].unflatten(1, (kv, hd))
    c = kv4.KV4Cache(1, kv, hd, 6, page, 3, 3)
    c.lens.copy_(ints([20, 4, 40]))  # the second holds fewer rows than it is given
    c.table.copy_(ints([[3, 1, -1], [2, -1, -1], [0, -1, 99]]))
    c.append(0, k, v, starts_of(lens))
    ko, vo = torch.full((T, kv, hd), 9.0, device="cuda"), torch.full((T, kv, hd), 9.0, device="cuda")
    c.read(0, ko, vo, starts_of(lens))
    want = quantised(k.float().cpu().numpy())
    got = ko.cpu().numpy()
    np.testing.assert_array_equal(got[:20], want[:20])
    np.testing.assert_array_equal(got[22:26], want[22:26])
    assert (got[20:22] == 9).all() and (got[26:] == 9).all()  # rows 31 .. 39 lie in pages -1 and 99
    c.append(0, k, v, starts_of(lens), ints([0, 7, -1]))  # slots that do not exist
    c.read(0, ko, vo, starts_of(lens))
    np.testing.assert_array_equal(ko.cpu().numpy()[:20], want[:20])


# ---- attention ---------------------------------------------------------------

def attend64(q, k, v, lens, scale, kind):
    """(output, tolerance): probabilities off by twice the scores' error
    (scale sum |q||k| (hd + 8) 2^-23), 2^-19 + |s| 2^-23 of the exponential and
    n 2^-23 of the sums, relative to sum p |v|; the result rounded once."""
    group, hd = q.shape[1] // k.shape[1], q.shape[2]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    at = 0
    for b, n in enumerate(lens):
        if n:
            for h in range(q.shape[1]):
                Q, K, V = q[b, h].double(), k[at:at + n, h // group].double(), v[at:at + n, h // group].double()
                s = K @ Q * scale
                ds = (K.abs() @ Q.abs()).max() * scale * (hd + 8) * 2.0 ** -23
                p = torch.softmax(s, 0)
                out[b, h] = p @ V
                tol[b, h] = (p @ V.abs()) * (2 * ds + 2 * s.abs().max() * 2.0 ** -23 + 2.0 ** -19 + n * 2.0 ** -23) + out[b, h].abs() * U[kind]
        at += n
    return out, tol


def run_attention(c, lens, q, scale, slot_ids=None):
    out = torch.full_like(q, float("nan"))
    c.attention(0, out, q, scale, slot_ids)
    return out


def held(c, lens, k, slot_ids=None):
    ko, vo = torch.empty(k.shape, device="cuda"), torch.empty(k.shape, device="cuda")
    c.read(0, ko, vo, starts_of(lens), slot_ids)
    return ko, vo


def check(got, want, tol):
    assert torch.isfinite(got).all()
    worst = ((got.double() - want).abs() - tol).max().item()
    assert worst <= 0, worst


@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("heads,kv,hd", [(4, 4, 32), (3, 3, 64), (6, 2, 64), (16, 2, 64), (32, 4, 128), (9, 1, 128), (34, 2, 32), (2, 2, 128)])
@pytest.mark.parametrize("kind", sorted(DT))
def test_attention(kind, heads, kv, hd, page):
    lens = [1, 0, 15, 16, 17, 100, 333, 2, 64, 1500]
    c, k, v = cache_with(lens, kv, hd, page, "fp32", 3)
    q = torch.randn(len(lens), heads, hd, device="cuda", generator=torch.Generator(device="cuda").manual_seed(4)).to(DT[kind])
    scale = 1 / math.sqrt(hd)
    out = run_attention(c, lens, q, scale)
    check(out, *attend64(q, *held(c, lens, k), lens, scale, kind))
    assert (out[1] == 0).all()
    assert torch.equal(out, run_attention(c, lens, q, scale))


@pytest.mark.parametrize("hd,heads,kv", [(128, 8, 2), (64, 4, 4), (32, 8, 1)])
def test_attention_of_long_sequences(hd, heads, kv):
    lens = [20011, 3, 9000, 40000]
    c, k, v = cache_with(lens, kv, hd, 64, "fp32", 5)
    for kind in sorted(DT):
        q = torch.randn(len(lens), heads, hd, device="cuda", generator=torch.Generator(device="cuda").manual_seed(6)).to(DT[kind])
        check(run_attention(c, lens, q, 0.11), *attend64(q, *held(c, lens, k), lens, 0.11, kind))


@pytest.mark.parametrize("batch", [127, 128, 129, 300, 1000])
@pytest.mark.parametrize("kind", sorted(DT))
def test_attention_of_many_sequences(kind, batch):
    """More entries than a block has threads to look their lengths up."""
    lens = np.random.RandomState(batch).randint(0, 90, batch).tolist()
    lens[batch // 2], lens[-1] = 2000, 700
    c, k, v = cache_with(lens, 1, 32, 16, "fp32", 12)
    q = torch.randn(batch, 3, 32, device="cuda", generator=torch.Generator(device="cuda").manual_seed(13)).to(DT[kind])
    out = run_attention(c, lens, q, 0.3)
    check(out, *attend64(q, *held(c, lens, k), lens, 0.3, kind))
    assert (out[[i for i, n in enumerate(lens) if n == 0]] == 0).all()


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("kind", ["fp16", "bf16"])
def test_attention_over_many_keys_of_about_equal_weight(kind, hd):
    """Sums of 30,000 values whose mean is what is left: in the norm, no more
    off than outputs rounded to their type (u / sqrt(3) at most) and a quarter
    of an fp16 rounding for all else, however many keys a block sums up."""
    n, kv, batch = 30000, 8, 24
    c = kv4.KV4Cache(1, kv, hd, n // 64 + 1, 64, 1)
    c.reserve(ints([n]))
    k, v = rows([n], kv, hd, "fp32", 50 + hd)
    c.append(0, k, v, starts_of([n]))
    ko, vo = (x.double().transpose(0, 1) for x in held(c, [n], k))
    q = (torch.randn(batch, kv, hd, device="cuda", generator=torch.Generator(device="cuda").manual_seed(51)) * 0.5).to(DT[kind])
    out = run_attention(c, [n], q, hd ** -0.5, ints([0] * batch))  # entries that read the same slot
    want = (torch.softmax(q.double().transpose(0, 1) @ ko.transpose(1, 2) * hd ** -0.5, -1) @ vo).transpose(0, 1)
    off = ((out.double() - want).norm() / want.norm()).item()
    assert off <= U[kind] / math.sqrt(3) + 2.0 ** -13, off


def test_a_pool_past_four_gigabytes():
    """Pages on both sides of 2^32 bytes: rows, attention, a fork's copy and compaction."""
    hd, kv, page, pages = 128, 8, 128, 27000
    c = kv4.KV4Cache(1, kv, hd, pages, page, 3, 4)
    assert c.pool[0].numel() > 1 << 32
    at = [26999, 5, 26500, 26214]  # 2^32 is in page 26214
    c.table[0].copy_(ints(at))
    c.refs[at] = 1
    c.lens[0] = 400
    k, v = rows([400], kv, hd, "fp32", 14)
    c.append(0, k, v, starts_of([400]))
    want_k, want_v = (torch.from_numpy(quantised(x.cpu().numpy())).cuda() for x in (k, v))
    c.refs[:5] = 1  # the first free pages: 6, and, once the others have moved, a few more
    c.fork(ints([0]), ints([2]))
    c.check()
    assert c.table[2].tolist() == [26999, 5, 26500, 6]
    c.refs[:5] = 0
    for _ in range(2):
        q = torch.randn(2, 2 * kv, hd, device="cuda")
        for slot in (0, 2):
            ko, vo = torch.empty_like(k), torch.empty_like(v)
            c.read(0, ko, vo, starts_of([400]), ints([slot]))
            assert torch.equal(ko, want_k) and torch.equal(vo, want_v)
        out = run_attention(c, [400, 400], q, 0.1, ints([0, 2]))
        check(out, *attend64(q, want_k.repeat(2, 1, 1), want_v.repeat(2, 1, 1), [400, 400], 0.1, "fp32"))
        c.compact()  # and once more as they lie then
    assert sorted(set(c.table.flatten().tolist())) == [-1, 0, 1, 2, 3, 4]


def test_attention_through_slots_strides_and_missing_pages():
    """Entries in another order than their slots, a slot that does not exist,
    a strided query, a page that does not exist (its keys are masked)."""
    lens, order, hd = [40, 33, 90], [4, 0, 2], 64
    c, k, v = cache_with(lens, 2, hd, 16, "fp32", 7, slots=5, order=order)
    ko, vo = held(c, lens, k, ints(order))
    flat = torch.randn(4, 4 * hd + 3, device="cuda")
    q = flat[:, 3:].unflatten(1, (4, hd))
    whole = torch.full((4, 4 * hd + 5), 3.0, device="cuda")
    out = whole[:, 1:1 + 4 * hd].unflatten(1, (4, hd))
    c.attention(0, out, q, 0.2, ints(order + [17]))
    want, tol = attend64(q, ko, vo, lens + [0], 0.2, "fp32")
    check(out, want, tol)
    assert (whole[:, 0] == 3).all() and (whole[:, 1 + 4 * hd:] == 3).all()
    c.table[2, 1] = -1        # rows 16 .. 31 of the last sequence
    c.table[2, 3] = 10 ** 6   # rows 48 .. 63
    c.attention(0, out, q, 0.2, ints(order + [-1]))
    keep = torch.ones(sum(lens), dtype=torch.bool, device="cuda")
    keep[73 + 16:73 + 32] = False
    keep[73 + 48:73 + 64] = False
    want, tol = attend64(q, ko[keep], vo[keep], [40, 33, 58, 0], 0.2, "fp32")
    check(out, want, tol)
    c.table[4].fill_(-1)      # a sequence none of whose pages exists
    c.attention(0, out, q, 0.2, ints(order + [-1]))
    assert (out[0] == 0).all()


def test_attention_scores_and_values_of_many_sizes():
    """Scores far apart, keys whose scores rise along the sequence, values and
    queries of very different magnitudes, groups that hold nothing but zeros."""
    hd, n = 64, 500
    g = torch.Generator(device="cuda").manual_seed(8)
    ramp = torch.linspace(0.05, 4, n, device="cuda")[:, None, None]
    for size_q, size_v in ((1.0, 1.0), (1e-6, 1e-4), (300.0, 3e4), (1.0, 1e-3)):
        c = kv4.KV4Cache(1, 1, hd, 40, 16, 1, 40)
        c.reserve(ints([n]))
        k = torch.randn(n, 1, hd, generator=g, device="cuda") * ramp / size_q
        v = torch.randn(n, 1, hd, generator=g, device="cuda") * size_v
        v[:200, :, :32] = 0.0
        v[100:110] *= 0.01
        c.append(0, k.clamp(-6e4, 6e4), v, starts_of([n]))
        q = torch.randn(1, 5, hd, generator=g, device="cuda") * size_q
        ko, vo = held(c, [n], k)
        check(run_attention(c, [n], q, 0.3), *attend64(q, ko, vo, [n], 0.3, "fp32"))


def scale_bits(c, table, n, hd, page, values):
    """The bits of the scales [n, kv, hd / 32] of one sequence's keys or values, as the pool holds them."""
    raw = c.pool[0].cpu().numpy().reshape(c.pool.shape[1], c.pool.shape[2], 2, -1)[:, :, int(values), page * hd // 2:]
    pairs = np.ascontiguousarray(raw).view(np.uint16).reshape(*raw.shape[:2], page, hd // 32, 2)
    return np.stack([pairs[table[t // page], :, t % page, :, 0] for t in range(n)])


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("kind", sorted(DT))
def test_attention_over_constant_groups_with_negative_scales(kind, hd):
    """A group's minimum is rounded to fp16, so that a constant group (0.3) may
    lie below it: its scale is then negative, or -0 (3e-8)."""
    n, page, kv = 200, 16, 2
    g = torch.Generator(device="cuda").manual_seed(hd)
    k, v = torch.randn(n, kv, hd, generator=g, device="cuda"), torch.randn(n, kv, hd, generator=g, device="cuda")
    for x in (k, v):
        x[::3, :, :32] = 0.3
        x[1::3, 0, hd - 32:] = 3e-8
        x[150:, 1, :32] = -0.7002  # and to the end
    c = kv4.KV4Cache(1, kv, hd, 20, page, 1, 20)
    c.reserve(ints([n]))
    c.append(0, k, v, starts_of([n]))
    for values in (False, True):
        bits = scale_bits(c, c.table[0].tolist(), n, hd, page, values)
        assert (bits[0, :, 0] > 0x8000).all() and bits[1, 0, -1] == 0x8000 and (bits[150:, 1, 0] > 0x8000).all()
    q = torch.randn(1, 3 * kv, hd, generator=g, device="cuda").to(DT[kind])
    check(run_attention(c, [n], q, 0.2), *attend64(q, *held(c, [n], k), [n], 0.2, kind))


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("kind", sorted(DT))
def test_attention_over_values_of_very_different_sizes(kind, hd):
    """Groups of 32 columns that reach fp16's limit beside ones of a
    thousandth, and single values at the limit among keys of a thousandth, which
    the softmax all but leaves out: every column is as good as its own values."""
    n, kv = 500, 2
    g = torch.Generator(device="cuda").manual_seed(40 + hd)
    k, v = (torch.randn(n, kv, hd, generator=g, device="cuda") for _ in range(2))
    size = torch.tensor([1e-3, 1.5e4, 1.0, 1e-5], device="cuda").repeat_interleave(32)[:hd]
    v *= size
    q = torch.randn(1, 2 * kv, hd, generator=g, device="cuda").to(DT[kind])
    for at in (0, 37, 250):  # keys that no query head of the group looks at
        v[at] = torch.randn(kv, hd, generator=g, device="cuda") * 2e4
        for h in range(kv):
            k[at, h] = -12 * q[0, 2 * h:2 * h + 2].float().mean(0)
    c = kv4.KV4Cache(1, kv, hd, 40, 16, 1, 40)
    c.reserve(ints([n]))
    c.append(0, k, v.clamp(-65504, 65504), starts_of([n]))
    want, tol = attend64(q, *held(c, [n], k), [n], 0.3, kind)
    # fp16 results below 2^-14 are rounded to multiples of 2^-24
    check(run_attention(c, [n], q, 0.3), want, tol + (2.0 ** -25 if kind == "fp16" else 0))


def test_attention_passes_nan_on():
    hd = 32
    c = kv4.KV4Cache(1, 2, hd, 4, 16, 1, 4)
    c.reserve(ints([20]))
    k = torch.randn(20, 2, hd, device="cuda")
    v = torch.randn(20, 2, hd, device="cuda")
    v[7, 1, 3] = float("nan")
    c.append(0, k, v, starts_of([20]))
    out = run_attention(c, [20], torch.randn(1, 4, hd, device="cuda"), 0.2)
    assert torch.isfinite(out[0, :2]).all() and torch.isnan(out[0, 2:]).all()


def test_attention_on_another_stream_and_in_a_graph():
    lens = [700, 4000]
    c, k, v = cache_with(lens, 2, 128, 64, "fp32", 9)
    q = torch.randn(2, 8, 128, device="cuda")
    want = run_attention(c, lens, q, 0.1)
    out = torch.empty_like(q)
    ws = torch.empty(max(1, kv4.attention_workspace_bytes(2, 8, 2, 128, c.table.shape[1], 64)), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(st):
        c.attention(0, out, q, 0.1, workspace=ws)
        st.synchronize()
        assert torch.equal(out, want)
        with torch.cuda.graph(graph, stream=st):
            c.attention(0, out, q, 0.1, workspace=ws)
        out.fill_(0)
        ws.fill_(255)  # any content
        graph.replay()
    st.synchronize()
    assert torch.equal(out, want)


# ---- pages ----------------------------------------------------------------------

class Model:
    """The page operations on lists."""

    def __init__(self, pages, slots, most, page):
        self.refs, self.table, self.lens = [0] * pages, [[-1] * most for _ in range(slots)], [0] * slots
        self.page, self.content, self.status = page, list(range(pages)), 0

    def _free(self):
        return [p for p, r in enumerate(self.refs) if r == 0]

    def reserve(self, slots, counts):
        need = [-(-(self.lens[s] + c) // self.page) - -(-self.lens[s] // self.page) for s, c in zip(slots, counts)]
        free = self._free()
        if sum(need) > len(free):
            self.status |= kv4.NO_PAGES
            return
        for s, c, n in zip(slots, counts, need):
            old = -(-self.lens[s] // self.page)
            for j in range(n):
                p = free.pop(0)
                self.table[s][old + j], self.refs[p] = p, 1
            self.lens[s] += c

    def fork(self, parents, children):
        free, before = self._free(), [self.lens[p] for p in parents]
        if sum(n % self.page != 0 for n in before) > len(free):
            self.status |= kv4.NO_PAGES
            return
        for p, c, n in zip(parents, children, before):
            full = n // self.page
            for j in range(full):
                self.table[c][j] = self.table[p][j]
                self.refs[self.table[p][j]] += 1
            if n % self.page:
                new = free.pop(0)
                self.refs[new], self.table[c][full] = 1, new
                self.content[new] = self.content[self.table[p][full]]
            self.lens[c] = n

    def free(self, slots):
        for s in slots:
            for j, p in enumerate(self.table[s]):
                if p >= 0:
                    self.refs[p] -= 1
                self.table[s][j] = -1
            self.lens[s] = 0

    def compact(self):
        n = sum(r > 0 for r in self.refs)
        holes = [p for p in range(n) if self.refs[p] == 0]
        movers = [p for p in range(n, len(self.refs)) if self.refs[p] > 0]
        to = dict(zip(movers, holes))
        for m, h in to.items():
            self.refs[h], self.refs[m], self.content[h] = self.refs[m], 0, self.content[m]
        self.table = [[to.get(p, p) for p in r] for r in self.table]

    def same(self, c):
        assert c.refs.tolist() == self.refs
        assert c.table.tolist() == self.table
        assert c.lens.tolist() == self.lens
        assert int(c.status) == self.status
        flat = c.pool.flatten(2)
        for l in range(flat.shape[0]):
            for p, r in enumerate(self.refs):
                if r:
                    assert (flat[l, p] == self.content[p] % 251).all(), (l, p)


@pytest.mark.parametrize("pages,slots,page", [(40, 9, 16), (300, 40, 32), (5000, 60, 16)])
def test_page_operations_follow_the_model(pages, slots, page):
    rng = np.random.RandomState(pages)
    most = max(4, pages // 8)
    c = kv4.KV4Cache(3, 2, 32, pages, page, slots, most)
    c.pool.copy_((torch.arange(pages, device="cuda") % 251).to(torch.uint8)[None, :, None, None, None].expand(c.pool.shape))
    m = Model(pages, slots, most, page)
    for step in range(60):
        empty = [s for s in range(slots) if m.lens[s] == 0]
        used = [s for s in range(slots) if m.lens[s]]
        what = rng.choice(["reserve", "reserve", "fork", "free", "compact"])
        if what == "reserve":
            pick = rng.permutation(slots)[:rng.randint(1, slots + 1)].tolist()
            counts = [int(rng.randint(0, min(3 * page, most * page - m.lens[s]) + 1)) for s in pick]
            c.reserve(ints(counts), ints(pick))
            m.reserve(pick, counts)
        elif what == "fork" and used and empty:
            n = rng.randint(1, len(empty) + 1)
            kids = rng.permutation(empty)[:n].tolist()
            folk = [int(rng.choice(used)) for _ in kids]
            c.fork(ints(folk), ints(kids))
            m.fork(folk, kids)
        elif what == "free" and used:
            gone = rng.permutation(slots)[:rng.randint(1, slots // 2 + 1)].tolist()
            c.free(ints(gone + gone[:1]))  # one named twice
            m.free(gone)
        else:
            c.compact()
            m.compact()
        m.same(c)
    m.free(range(slots))
    c.free(ints(list(range(slots))))
    m.same(c)
    assert int(c.refs.sum()) == 0


def test_page_operations_that_cannot_be_carried_out_change_nothing():
    c = kv4.KV4Cache(1, 1, 32, 4, 16, 4, 3)
    c.reserve(ints([20, 5]), ints([0, 2]))
    before = [t.clone() for t in (c.refs, c.table, c.lens, c.pool)]

    def unchanged(bit):
        for t, u in zip((c.refs, c.table, c.lens, c.pool), before):
            assert torch.equal(t, u)
        assert int(c.status) == bit
        with pytest.raises(FmlError):
            c.check()
        c.check()

    c.reserve(ints([1, 40]), ints([1, 3]))       # five pages, one is free
    unchanged(kv4.NO_PAGES)
    c.reserve(ints([1, 40]), ints([1, 0]))       # 60 rows in a table row of 48
    unchanged(kv4.ROW_FULL)
    c.reserve(ints([1, 1]), ints([1, 1]))        # named twice
    unchanged(kv4.BAD_SLOT)
    c.reserve(ints([1, 1]), ints([1, 4]))
    unchanged(kv4.BAD_SLOT)
    c.fork(ints([0, 2]), ints([1, 3]))           # two pages in use, one is free
    unchanged(kv4.NO_PAGES)
    c.fork(ints([0]), ints([2]))                 # a child that holds rows
    unchanged(kv4.BAD_SLOT)
    c.fork(ints([0, 0]), ints([1, 1]))           # named twice
    unchanged(kv4.BAD_SLOT)
    c.fork(ints([0, -1]), ints([1, 3]))
    unchanged(kv4.BAD_SLOT)
    c.fork(ints([0]), ints([1]))
    c.check()
    assert c.refs.tolist() == [2, 1, 1, 1] and c.table[1].tolist() == [0, 3, -1]


def test_a_fork_of_thousands_is_refused_whole():
    """One child among several thousand holds rows, or is named twice, or the
    pages run out: the block that settles a fork takes its entries in turns,
    and all of its threads must come to the same end."""
    n = 2500
    c = kv4.KV4Cache(1, 1, 32, n + 8, 16, 2 * n + 2, 2)
    c.reserve(ints([20, 16]), ints([0, 1]))
    before = [t.clone() for t in (c.refs, c.table, c.lens, c.pool)]

    def refused(parents, children, bit):
        c.fork(ints(parents), ints(children))
        for t, u in zip((c.refs, c.table, c.lens, c.pool), before):
            assert torch.equal(t, u)
        assert int(c.status) == bit
        c.status.zero_()

    kids = list(range(2, n + 2))
    for _ in range(20):
        for at in (0, 31, 1023, 1024, n - 1):
            refused([0] * n, kids[:at] + [1] + kids[at + 1:], kv4.BAD_SLOT)      # a child that holds rows
            refused([0] * n, kids[:at] + [kids[at - 1]] + kids[at + 1:], kv4.BAD_SLOT)  # a child named twice
            refused([0] * n, kids[:at] + [2 * n + 2] + kids[at + 1:], kv4.BAD_SLOT)  # no such slot
        refused([0] * (n + 6), list(range(2, n + 8)), kv4.NO_PAGES)  # one page short
    c.fork(ints([0] * n), ints(kids))
    c.check()
    assert c.refs[:3].tolist() == [n + 1, 1, 1] and int(c.refs.sum()) == n + 1 + 2 + n
    assert c.table[2:n + 2, 1].tolist() == list(range(3, n + 3))
    # the same of a reserve: more pages than are free, and than there are at all
    before = [t.clone() for t in (c.refs, c.table, c.lens, c.pool)]
    free = list(range(n + 2, 2 * n + 2))
    for rows_each in (1, 32) * 20:
        c.reserve(ints([rows_each] * n), ints(free))
        for t, u in zip((c.refs, c.table, c.lens, c.pool), before):
            assert torch.equal(t, u)
        assert int(c.status) == kv4.NO_PAGES
        c.status.zero_()


def test_an_append_behind_a_refused_reserve_writes_nothing():
    """A full pool, sequences that share their last full page: the rows of a
    step that finds no page must not land on the newest rows there are."""
    hd, kv, L, page = 64, 2, 2, 16
    c = kv4.KV4Cache(L, kv, hd, 4, page, 4, 4)
    k, v = rows([54], kv, hd, "fp32", 21)

    def append(at, n, ids):
        b = len(ids)
        for l in range(L):
            c.append(l, k[at:at + n].repeat(b, 1, 1), v[at:at + n].repeat(b, 1, 1), starts_of([n] * b), ints(ids))

    c.reserve(ints([32]), ints([2]))
    append(0, 32, [2])
    c.fork(ints([2]), ints([0]))
    c.reserve(ints([20]), ints([1]))
    append(32, 20, [1])
    c.check()
    before = [t.clone() for t in (c.refs, c.table, c.lens, c.pool)]
    q = torch.randn(3, 4, hd, device="cuda")
    out = torch.empty_like(q)
    c.attention(1, out, q, 0.2, ints([0, 1, 2]))
    c.reserve(ints([1, 1, 1]), ints([0, 1, 2]))  # two pages more, none is free
    append(52, 1, [0, 1, 2])
    again = torch.empty_like(q)
    c.attention(1, again, q, 0.2, ints([0, 1, 2]))
    for t, u in zip((c.refs, c.table, c.lens, c.pool), before):
        assert torch.equal(t, u)
    assert torch.equal(out, again)
    # a refusal for another reason, the row of a slot that is not in it is written
    c.reserve(ints([1]), ints([1]))
    c.reserve(ints([1, 99]), ints([0, 2]))
    append(52, 1, [0, 1, 2])
    assert c.lens.tolist() == [32, 21, 32, 0] and torch.equal(c.pool[:, :2], before[3][:, :2])
    ko, vo = torch.empty(21, kv, hd, device="cuda"), torch.empty(21, kv, hd, device="cuda")
    c.read(1, ko, vo, starts_of([21]), ints([1]))
    np.testing.assert_array_equal(vo.cpu().numpy(), quantised(v[32:53].cpu().numpy()))
    with pytest.raises(FmlError):
        c.check()
    # a slot that was refused goes on: freed and filled anew, and where its rows end
    c.reserve(ints([1, 9]), ints([0, 7]))
    c.free(ints([0, 1]))
    c.reserve(ints([5, 3]), ints([0, 2]))
    for l in range(L):
        c.append(l, k[:8], v[:8], starts_of([5, 3]), ints([0, 2]))
    for slot, n, want in ((0, 5, v[:5]), (2, 3, v[5:8]), (2, 35, torch.cat([v[:32], v[5:8]]))):
        ko, vo = torch.empty(n, kv, hd, device="cuda"), torch.empty(n, kv, hd, device="cuda")
        c.read(0, ko, vo, starts_of([n]), ints([slot]))
        np.testing.assert_array_equal(vo.cpu().numpy(), quantised(want.cpu().numpy()))
    # two reserves before their rows; rows written again after check() has told of a refusal
    with pytest.raises(FmlError):
        c.check()
    c.reserve(ints([2]), ints([0]))
    c.reserve(ints([3]), ints([0]))
    c.append(0, k[10:15], v[10:15], starts_of([5]), ints([0]))
    c.reserve(ints([99]), ints([0]))
    with pytest.raises(FmlError):
        c.check()
    c.append(0, k[20:24], v[20:24], starts_of([4]), ints([0]))
    ko, vo = torch.empty(10, kv, hd, device="cuda"), torch.empty(10, kv, hd, device="cuda")
    c.read(0, ko, vo, starts_of([10]), ints([0]))
    np.testing.assert_array_equal(vo.cpu().numpy(), quantised(torch.cat([v[:5], v[10:11], v[20:24]]).cpu().numpy()))


def test_forked_sequences_go_their_own_ways():
    """A prompt forked in the middle of a page: both append, both attend to
    their own rows, and compaction after the parent's end changes nothing."""
    hd, kv, L = 64, 2, 2
    c = kv4.KV4Cache(L, kv, hd, 64, 16, 4, 8)
    k, v = rows([40], kv, hd, "fp32", 11)
    c.reserve(ints([30]), ints([3]))
    for l in range(L):
        c.append(l, k[:30], v[:30], starts_of([30]), ints([3]))
    c.fork(ints([3, 3]), ints([1, 0]))
    c.reserve(ints([10, 10, 10]), ints([3, 1, 0]))
    for l in range(L):
        new_k = torch.cat([k[30:], k[30:] + 1, k[30:] - 1])
        new_v = torch.cat([v[30:], v[30:] * 2, v[30:] * 3])
        c.append(l, new_k, new_v, starts_of([10, 10, 10]), ints([3, 1, 0]))
    c.free(ints([3]))
    c.compact()
    c.check()
    used = int((c.refs > 0).sum())
    assert (c.refs[:used] > 0).all() and used == 5  # one full page shared, two of their own each
    q = torch.randn(2, 4, hd, device="cuda")
    for l in range(L):
        out = torch.empty_like(q)
        c.attention(l, out, q, 0.2, ints([1, 0]))
        kk = torch.cat([k[:30], k[30:] + 1, k[:30], k[30:] - 1])
        vv = torch.cat([v[:30], v[30:] * 2, v[:30], v[30:] * 3])
        ko, vo = (torch.from_numpy(quantised(x.cpu().numpy())).cuda() for x in (kk, vv))
        check(out, *attend64(q, ko, vo, [40, 40], 0.2, "fp32"))


def test_refusals():
    c = kv4.KV4Cache(1, 2, 64, 4, 16, 2, 2)
    x = torch.zeros(2, 2, 64, device="cuda")
    s = starts_of([1, 1])
    with pytest.raises(FmlError):
        kv4.KV4Cache(1, 2, 48, 4, 16, 2, 2)
    with pytest.raises(FmlError):
        kv4.KV4Cache(1, 2, 64, 4, 24, 2, 2)
    with pytest.raises(FmlError):
        c.append(0, x[:, :1], x[:, :1], s)
    with pytest.raises(FmlError):
        c.append(0, x, x.half(), s)
    with pytest.raises(FmlError):
        c.append(0, x.double(), x.double(), s)
    with pytest.raises(FmlError):
        c.append(0, x, x, s.long())
    with pytest.raises(FmlError):
        c.append(0, x, x, s, ints([0]))
    with pytest.raises(FmlError):
        c.attention(0, x, torch.zeros(2, 3, 64, device="cuda"), 0.1)  # out of another shape
    q = torch.zeros(2, 3, 64, device="cuda")
    with pytest.raises(FmlError):
        c.attention(0, q, q, 0.1)  # three query heads over two
    with pytest.raises(FmlError):
        c.fork(ints([0]), ints([0, 1]))
    big = kv4.KV4Cache(1, 8, 64, 4, 128, 1, 4096)
    q = torch.zeros(1, 8, 64, device="cuda")
    if kv4.attention_workspace_bytes(1, 8, 8, 64, 4096, 128):
        with pytest.raises(FmlError):
            big.attention(0, q, q, 0.1, workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
