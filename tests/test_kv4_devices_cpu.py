"""The 4-bit cache's and the packed attention's Python entry points: every
tensor, a caller's workspace too, is on one GPU, the call is made with that GPU
current, on its stream, and row strides fit the C ABI's 32 bits.  Tensors are stand-ins, and the library's calls are
noted instead of made, so that no GPU is needed and none is reached."""
import contextlib

import pytest
import torch

from freeml_b200 import FmlError, kv4, matrix_ops


class Stand:
    """What the checks ask of a CUDA tensor."""

    def __init__(self, shape, dtype, device=0, stride=None, dense=True):
        self.shape, self.dtype, self.at, self.dense = tuple(shape), dtype, device, dense
        self.steps = stride or [int(torch.tensor(self.shape[i + 1:]).prod()) for i in range(len(self.shape))]
        self.device = torch.device("cuda", device) if device >= 0 else torch.device("cpu")
        self.is_cuda = device >= 0

    def dim(self):
        return len(self.shape)

    def stride(self):
        return tuple(self.steps)

    def is_contiguous(self):
        return self.dense

    def data_ptr(self):
        return 0x10000

    def get_device(self):
        return self.at

    def numel(self):
        return int(torch.tensor(self.shape).prod())

    def element_size(self):
        return torch.empty(0, dtype=self.dtype).element_size()


def i32(*shape):
    return Stand(shape, torch.int32)


def tensors():
    """Every argument that is a tensor, of shapes that go together."""
    f = lambda: Stand((3, 4, 64), torch.float32)  # noqa: E731
    return dict(pool=Stand((8, 2, 16, 80), torch.uint8), pools=Stand((5, 8, 2, 16, 80), torch.uint8), table=i32(4, 6), lens=i32(4),
                ids=i32(2), starts=i32(3), k=Stand((3, 2, 64), torch.float32), v=Stand((3, 2, 64), torch.float32), kept=i32(4),
                q=Stand((2, 4, 64), torch.float32), out=Stand((2, 4, 64), torch.float32), refs=i32(8), counts=i32(2), status=i32(1),
                kids=i32(2), pq=f(), po=f(), work=Stand((1 << 24,), torch.uint8))


CALLS = {
    "append": ("pool table lens k v starts ids kept", lambda t: kv4.append(t["pool"], t["table"], t["lens"], t["k"], t["v"], t["starts"], t["ids"], t["kept"])),
    "read": ("pool table lens k v starts ids", lambda t: kv4.read(t["k"], t["v"], t["pool"], t["table"], t["lens"], t["starts"], t["ids"])),
    "attention": ("pool table lens q out ids work", lambda t: kv4.attention(t["out"], t["q"], t["pool"], t["table"], t["lens"], 0.1, t["ids"], t["work"])),
    "reserve": ("refs table lens counts status ids work kept", lambda t: kv4.reserve(t["refs"], t["table"], t["lens"], t["counts"], 16, t["status"], t["ids"], t["work"], t["kept"])),
    "fork": ("pools refs table lens ids kids status work", lambda t: kv4.fork(t["pools"], t["refs"], t["table"], t["lens"], t["ids"], t["kids"], t["status"], t["work"])),
    "free": ("refs table lens ids status", lambda t: kv4.free(t["refs"], t["table"], t["lens"], t["ids"], t["status"])),
    "compact": ("pools refs table work", lambda t: kv4.compact(t["pools"], t["refs"], t["table"], t["work"])),
    "packed": ("po pq k v starts", lambda t: matrix_ops.attention_packed(t["po"], t["pq"], t["k"], t["v"], t["starts"], 0.1, mode=1)),
}


@pytest.fixture
def made(monkeypatch):
    """The calls made: name, the GPU that was current, the stream."""
    log, current = [], [0]

    @contextlib.contextmanager
    def device(d):
        before, current[0] = current[0], getattr(d, "index", d)
        yield
        current[0] = before

    note = lambda name, *args: log.append((name, current[0], args[-1], args))  # noqa: E731
    monkeypatch.setattr(kv4, "call", note)
    monkeypatch.setattr(matrix_ops, "call", note)
    monkeypatch.setattr(kv4, "_raw_stream", lambda d: 100 + d)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", device)
    return log


@pytest.mark.parametrize("name", sorted(CALLS))
def test_the_tensors_gpu_is_made_current(name, made):
    uses, run = CALLS[name]
    run(tensors())
    t = tensors()
    for x in t.values():
        x.at, x.device = 1, torch.device("cuda", 1)
    run(t)
    assert [m[1:3] for m in made] == [(0, 100), (1, 101)]


@pytest.mark.parametrize("name", sorted(CALLS))
def test_tensors_of_another_device_are_refused(name, made):
    uses, run = CALLS[name]
    for which in uses.split():
        for elsewhere in (1, -1):
            t = tensors()
            t[which] = Stand(t[which].shape, t[which].dtype, elsewhere)
            with pytest.raises(FmlError):
                run(t)
    assert not made


@pytest.mark.parametrize("name", [n for n in sorted(CALLS) if "work" in CALLS[n][0]])
def test_a_workspace_with_gaps_is_refused(name, made):
    t = tensors()
    t["work"] = Stand((1 << 20, 2), torch.float32, stride=[64, 1], dense=False)
    with pytest.raises(FmlError):
        CALLS[name][1](t)
    assert not made


@pytest.mark.parametrize("name,which,heads", [("append", "k", 2), ("append", "v", 2), ("read", "k", 2), ("attention", "q", 4),
                                              ("attention", "out", 4), ("packed", "pq", 4), ("packed", "po", 4), ("packed", "k", 2)])
def test_rows_too_far_apart_are_refused(name, which, heads, made):
    """A stride of 2^32 elements and more would be cut to its low 32 bits."""
    t = tensors()
    for stride in (1 << 32, (1 << 32) + 64 * heads):
        t[which] = Stand(t[which].shape, t[which].dtype, stride=[stride, 64, 1])
        with pytest.raises(FmlError):
            CALLS[name][1](t)
    assert not made
    t[which] = Stand(t[which].shape, t[which].dtype, stride=[(1 << 32) - 64, 64, 1])
    CALLS[name][1](t)
    assert (1 << 32) - 64 in made[0][3]


def test_a_single_row_has_no_stride(made):
    """One row of a tensor whose rows lie anywhere."""
    t = tensors()
    t["q"], t["out"] = (Stand((1, 4, 64), torch.float32, stride=[s, 64, 1]) for s in ((1 << 32) + 64, 256))
    t["ids"] = i32(1)
    CALLS["attention"][1](t)
    assert made[0][3][3:5] == (256, 256)
