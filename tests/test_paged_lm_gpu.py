"""PagedLM (freeml_b200/paged_lm.py): the packed prompt attention, the 4-bit
cache, its attention and its page operations together, against the PyTorch
restatement -- prompts in fp32, decoded rows over the values that the cache
holds (read back from it, so that a code on the edge between two values is the
same on both sides).  The bound is the logits': 1e-3 absolute and relative."""
import math

import numpy as np
import pytest
import torch

from freeml_b200 import FmlError, _lib
from freeml_b200.lm import NanoLLMShape, random_params
from freeml_b200.paged_lm import PagedLM
from tests import torch_ref

pytestmark = pytest.mark.gpu

SHAPES = [NanoLLMShape(256, 128, 128, 4, 4), NanoLLMShape(97, 200, 128, 2, 3)]


def prompts_of(shape, lens, seed=0):
    rng = np.random.RandomState(seed)
    return [rng.randint(0, shape.vocab, n).tolist() for n in lens]


def cached(lm, slot):
    """Per layer, the keys and values [rows, heads, hd] that a slot's cache stands for."""
    n, s = lm.length[slot], lm.shape
    starts, ids = lm._ints([0, n]), lm._ints([slot])
    out = []
    for layer in range(s.n_layer):
        k, v = (torch.empty(n, s.n_head, lm.hd, device="cuda") for _ in range(2))
        lm.cache.read(layer, k, v, starts, ids)
        out.append((k.double(), v.double()))
    return out


def step64(lm, token, position, cache):
    """The logits after one token whose rows `cache` holds already."""
    ln = lambda x, g: torch_ref._layernorm(x, g.double())  # noqa: E731
    d, H = lm.shape.d_model, lm.shape.n_head
    x = lm.tok[token].double() + lm.pos[position].double()
    for w, (k, v) in zip(lm.layers, cache):
        q = (ln(x, w["ln0"]) @ w["qkv"].double())[:d].view(H, lm.hd)
        p = torch.softmax(torch.einsum("hd,khd->hk", q, k) / math.sqrt(lm.hd), -1)
        x = x + torch.einsum("hk,khd->hd", p, v).reshape(d) @ w["proj"].double().t()
        x = x + torch.nn.functional.gelu(ln(x, w["ln1"]) @ w["fc"].double()) @ w["mlp"].double()
    return ln(x, lm.lnf) @ lm.tok.double().t()


@pytest.mark.parametrize("shape", SHAPES)
def test_ragged_prompts_then_steps(shape):
    torch.backends.cuda.matmul.allow_tf32 = False
    params = random_params(shape, 3)
    lm = PagedLM(shape, params, pages=60, page_size=16, slots=5)
    prompts = prompts_of(shape, [1, 40, 17, 90])
    slots = [4, 0, 3, 1]
    logits = lm.prefill(prompts, slots)
    for row, p in zip(logits, prompts):
        want = torch_ref.forward(params, shape.vocab, shape.context, shape.d_model, shape.n_head, shape.n_layer, p,
                                 len(p) - 1, 1)[0]
        torch.testing.assert_close(row, want, rtol=1e-3, atol=1e-3)
    tokens = logits.argmax(-1).tolist()
    for _ in range(20):
        at = [lm.length[i] for i in slots]
        got = lm.step(tokens, slots)
        for row, slot, token, position in zip(got, slots, tokens, at):
            want = step64(lm, token, position, cached(lm, slot))
            torch.testing.assert_close(row.double(), want, rtol=1e-3, atol=1e-3)
        tokens = got.argmax(-1).tolist()
    lm.cache.check()


def test_forks_continue_as_their_parent_does():
    shape = SHAPES[0]
    lm = PagedLM(shape, random_params(shape, 5), pages=40, page_size=16, slots=6)
    logits = lm.prefill(prompts_of(shape, [37, 20], 1), [2, 5])
    lm.fork([2, 2, 5], [0, 1, 3])
    token = int(logits[0].argmax())
    # the same token for the parent and its first child, another for the second
    out = lm.step([token, token, (token + 1) % shape.vocab, 7], [2, 0, 1, 3])
    torch.testing.assert_close(out[0], out[1], rtol=1e-6, atol=1e-6)
    assert not torch.allclose(out[0], out[2], rtol=1e-3, atol=1e-3)
    before = [cached(lm, i) for i in (0, 1, 3)]
    lm.free([2, 5])
    lm.compact()
    lm.cache.check()
    used = int((lm.cache.refs > 0).sum())
    assert (lm.cache.refs[:used] > 0).all() and (lm.cache.refs[used:] == 0).all()
    for i, old in zip((0, 1, 3), before):
        for (k, v), (ko, vo) in zip(cached(lm, i), old):
            assert torch.equal(k, ko) and torch.equal(v, vo)
    got = lm.step([3, 3, 3], [0, 1, 3])
    for row, slot in zip(got, (0, 1, 3)):
        torch.testing.assert_close(row.double(), step64(lm, 3, lm.length[slot] - 1, cached(lm, slot)), rtol=1e-3, atol=1e-3)


def state_of(lm):
    c = lm.cache
    return [t.clone() for t in (c.refs, c.table, c.lens, c.pool)] + [list(lm.length)]


def unchanged(lm, before):
    now = state_of(lm)
    return all(torch.equal(a, b) for a, b in zip(now[:4], before[:4])) and now[4] == before[4]


def test_steps_and_forks_that_find_no_page():
    """A step on a full cache raises and changes nothing, not even the full
    last page that two forks share, and goes on once there is room."""
    shape = SHAPES[0]
    params = random_params(shape, 7)
    lm = PagedLM(shape, params, pages=6, page_size=16, slots=5)
    free = PagedLM(shape, params, pages=40, page_size=16, slots=5)
    prompts = prompts_of(shape, [32, 47, 3], 2)
    for one in (lm, free):
        one.prefill(prompts, [0, 1, 4])
        one.fork([0], [2])  # two full pages, shared
    assert int((lm.cache.refs == 0).sum()) == 0
    before = state_of(lm)
    for _ in range(2):
        with pytest.raises(FmlError):
            lm.step([1, 2, 3], [0, 1, 2])
        assert unchanged(lm, before)
    with pytest.raises(FmlError):
        lm.fork([1], [3])  # 47 rows: a page in use would be copied
    assert unchanged(lm, before)
    # prompts read no cache: their logits are right, their slot stays empty, and check() tells
    logits = lm.prefill([prompts[2]], [3])
    torch.testing.assert_close(logits, free.prefill([prompts[2]], [3]))
    assert unchanged(lm, before)
    with pytest.raises(FmlError):
        lm.step([1], [3])
    with pytest.raises(FmlError):
        lm.cache.check()
    lm.cache.check()
    # a refusal that nobody has asked about yet is not a later step's
    lm.cache.reserve(lm._ints([1]), lm._ints([9]))
    torch.testing.assert_close(lm.step([5], [1]), free.step([5], [1]))
    for one in (lm, free):
        one.free([4, 1])
    torch.testing.assert_close(lm.step([1, 2], [0, 2]), free.step([1, 2], [0, 2]))
    assert lm.length == [33, 0, 33, 0, 0] and lm.cache.lens.tolist() == lm.length
    with pytest.raises(FmlError):
        lm.cache.check()


def test_slots_that_are_not_as_they_should_be():
    """Refused on the host: the device's lengths and the host's stay the same."""
    shape = SHAPES[0]
    lm = PagedLM(shape, random_params(shape, 8), pages=20, page_size=16, slots=4)
    lm.prefill(prompts_of(shape, [20, 5], 3), [0, 1])
    before = state_of(lm)
    for bad in (lambda: lm.prefill([[1], [2]], [2, 2]), lambda: lm.prefill([[1]], [4]), lambda: lm.prefill([[1]], [-1]),
                lambda: lm.prefill([[1]], [2, 3]), lambda: lm.step([1, 2], [0, 0]), lambda: lm.step([1], [-4]),
                lambda: lm.step([1], [7]), lambda: lm.step([1, 2], [0]), lambda: lm.step([1], [0, 1]),
                lambda: lm.fork([0], [1]), lambda: lm.fork([0, 0], [2, 2]), lambda: lm.fork([0], [-1]),
                lambda: lm.fork([-4], [2]), lambda: lm.fork([0], [2, 3]), lambda: lm.fork([0, 1], [2]),
                lambda: lm.free([4]), lambda: lm.free([0, -3])):
        with pytest.raises(FmlError):
            bad()
        assert unchanged(lm, before)
    lm.cache.check()
    lm.free([0, 0])  # named twice, freed once
    assert lm.length == [0, 5, 0, 0] and lm.cache.lens.tolist() == lm.length
    lm.cache.check()


def test_refusals_and_the_example():
    from freeml_b200 import paged_lm
    shape = SHAPES[0]
    lm = PagedLM(shape, random_params(shape, 0), pages=4, page_size=16, slots=2)
    with pytest.raises(FmlError):
        lm.step([1], [0])
    with pytest.raises(FmlError):
        lm.prefill([[]], [0])
    with pytest.raises(FmlError):
        PagedLM(shape, torch.zeros(5, device="cuda"), pages=4)
    lm.prefill([[1] * 60], [0])
    lm.prefill([[1] * 10], [1])  # no page is left: noted on the device
    with pytest.raises(FmlError):
        lm.cache.check()
    before = _lib.launch_count()
    paged_lm.main()
    assert _lib.launch_count() > before
