"""Which stream and device the Python forms launch on, and what becomes of the memory they allocate, without a GPU:
tensors that say they are on a device, and a library that notes its calls."""
from __future__ import annotations

from contextlib import contextmanager

import pytest
import torch

from opfoundry_amd import dsa

DEV = 1
CURRENT = 5000                  # the current stream of device d is CURRENT + d


class Dev(torch.Tensor):
    """A host tensor that says it is on device DEV, and notes the streams it is marked for."""
    is_cuda = True
    marked = {}

    def get_device(self):
        return DEV

    def record_stream(self, stream):
        Dev.marked.setdefault(self.data_ptr(), []).append(stream.cuda_stream)


class FakeStream:
    def __init__(self, handle, device=None):
        self.cuda_stream = handle

    def wait_stream(self, other):
        waits.append((self.cuda_stream, other.cuda_stream))


waits = []


class Library:
    def __init__(self, state):
        self.state, self.launches = state, []

    def __getattr__(self, name):
        def call(*args):
            if name.endswith("_workspace_size"):
                args[1]._obj.value = 4096
            else:
                self.launches.append((name, self.state["device"], args))
            return 0
        return call


@pytest.fixture
def lib(monkeypatch):
    state = {"device": DEV}
    library = Library(state)

    @contextmanager
    def device(d):
        before, state["device"] = state["device"], d
        yield
        state["device"] = before

    Dev.marked = {}
    waits.clear()
    monkeypatch.setattr(dsa, "load_library", lambda: library)
    monkeypatch.setattr(dsa, "_current_device", lambda: state["device"])
    monkeypatch.setattr(dsa, "_raw_stream", lambda d: CURRENT + d)
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch.cuda, "ExternalStream", FakeStream)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda d=None: FakeStream(CURRENT + state["device"] if d is None else CURRENT + d))
    return library


def t(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype).as_subclass(Dev)


def i32(*v):
    return torch.tensor(v, dtype=torch.int32).as_subclass(Dev)


U8, F32 = torch.uint8, torch.float32


def mx(rows):
    return t(rows, 512, dtype=U8), t(rows, 16, dtype=U8), t(rows, 64)


# form -> (the call, the library's entry, whether it has a workspace)
FORMS = {
    "mla_decode": (lambda **k: dsa.mla_decode(t(2, 1, 16, 576), t(64, 400, dtype=U8), i32(*range(8)).view(2, 1, 4), 0.1,
                                              seq_lens=i32(4, 4), **k), True),
    "mla_decode_csr": (lambda **k: dsa.mla_decode_csr(t(2, 16, 576), t(64, 576), i32(0, 2, 4), i32(0, 1, 2, 3), 0.1, max_kv_len=2, **k), True),
    "csr_plan": (lambda **k: dsa.csr_plan(i32(0, 2, 4), 2, 1, 16, 2, **k), True),
    "mla_decode_mxfp8": (lambda **k: dsa.mla_decode_mxfp8(t(2, 16, 512, dtype=U8), t(2, 16, 16, dtype=U8), t(2, 16, 64), *mx(64),
                                                          i32(0, 2, 4), i32(0, 1, 2, 3), 0.1, max_kv_len=2, **k), True),
    "mla_combine": (lambda **k: dsa.mla_combine(t(3, 2, 16, 512, dtype=F32), t(3, 2, 16, dtype=F32), **k), False),
    "mla_prefill": (lambda **k: dsa.mla_prefill(t(2, 16, 576), t(64, 656, dtype=U8), i32(*range(8)).view(2, 4), 0.1, **k), True),
    "mla_prefill_v4": (lambda **k: dsa.mla_prefill_v4(t(2, 16, 512), t(64, 512), t(64, 512), None, i32(0, 1, 2), i32(0, 1), i32(0, 1, 2),
                                                      i32(0, 1), 0.1, max_rows=2, **k), True),
    "mla_prefill_v4_fp8": (lambda **k: dsa.mla_prefill_v4_fp8(t(2, 16, 512, dtype=U8), t(2, 16, 64), t(64, 512, dtype=U8), t(64, 64),
                                                              t(64, 512, dtype=U8), t(64, 64), None, i32(0, 1, 2), i32(0, 1), i32(0, 1, 2),
                                                              i32(0, 1), 0.1, max_rows=2, **k), True),
    "quantize_kv_fp8": (lambda **k: dsa.quantize_kv_fp8(t(3, 576), **k), False),
    "topk_indices": (lambda **k: dsa.topk_indices(t(2, 8, dtype=F32), 4, **k), False),
    "indexer_scores": (lambda **k: dsa.indexer_scores(t(2, 1, 4, 128), t(2, 1, 4, dtype=F32), t(64, 128), i32(4, 4), n_cols=4, **k), False),
    "mla_chunk": (lambda **k: dsa.mla_chunk(t(3, 16, 576), t(64, 400, dtype=U8), i32(0, 3), i32(9), 0.1, **k), True),
    "kv_read": (lambda **k: dsa.kv_read(t(64, 400, dtype=U8), i32(0, 3), i32(9), 3, **k), False),
}


def results(r):
    return [x for x in (r if isinstance(r, tuple) else (r,)) if isinstance(x, torch.Tensor)]


@pytest.mark.parametrize("form", FORMS)
def test_the_current_stream_of_the_tensors_device(lib, form):
    call, _ = FORMS[form]
    lib.state["device"] = DEV
    call()
    (name, device, args), = lib.launches
    assert device == DEV and args[-1] == CURRENT + DEV
    assert not Dev.marked and not waits
    # the same with another device current
    lib.launches.clear()
    lib.state["device"] = 0
    call()
    (name, device, args), = lib.launches
    assert device == DEV and args[-1] == CURRENT + DEV, "launched on another device, or on its stream"
    assert lib.state["device"] == 0
    assert not Dev.marked and not waits


@pytest.mark.parametrize("current", [DEV, 0])
@pytest.mark.parametrize("form", FORMS)
def test_memory_used_on_another_stream_is_marked_for_it(lib, form, current):
    """Output, LSE and workspace that a call allocates for stream 77: the stream waits for the current one's earlier work,
    and the allocator is told of it."""
    call, sized = FORMS[form]
    lib.state["device"] = current
    made = results(call(stream=77))
    (name, device, args), = lib.launches
    assert device == DEV and args[-1] == 77
    assert waits and set(waits) == {(77, CURRENT + DEV)}
    assert made and all(Dev.marked.get(x.data_ptr()) == [77] for x in made), "an output may be handed out while the call runs"
    if sized:
        ws = args[-3] if isinstance(args[-3], int) and args[-2] >= 4096 else None
        assert ws and Dev.marked.get(ws) == [77], "the workspace may be handed out while the call runs"


def test_a_copy_of_rows_is_marked(lib):
    """Rows that no one stride reaches are copied on the current stream, which the call's stream waits for."""
    src = t(3, 2, 640)[:, :, :576].transpose(0, 1)
    dsa.quantize_kv_fp8(src, stream=77)
    (name, device, args), = lib.launches
    assert args[0] != src.data_ptr() and Dev.marked.get(args[0]) == [77]


@pytest.mark.parametrize("form", ["mla_decode", "mla_prefill", "mla_decode_csr", "mla_decode_mxfp8", "mla_prefill_v4", "mla_chunk"])
def test_a_workspace_that_is_not_dense_or_elsewhere_is_refused(lib, form):
    call, _ = FORMS[form]
    for ws in (t(1, dtype=U8).expand(1 << 16), torch.zeros(1 << 16, dtype=U8)):
        with pytest.raises(ValueError):
            call(workspace=ws)
    assert not lib.launches
    call(workspace=t(1 << 16, dtype=U8))
    assert len(lib.launches) == 1


def test_tensors_of_another_device_are_refused(lib):
    q, kv, idx, sl = t(2, 1, 16, 576), t(64, 400, dtype=U8), i32(*range(8)).view(2, 1, 4), i32(4, 4)
    host = lambda x: torch.zeros(x.shape, dtype=x.dtype)                                          # noqa: E731
    for bad in (dict(kv_cache=host(kv)), dict(out=torch.zeros((2, 1, 16, 512), dtype=torch.bfloat16)), dict(lse=torch.zeros((2, 1, 16))),
                dict(indices=host(idx)), dict(seq_lens=host(sl)), dict(q=host(q))):
        with pytest.raises(ValueError):
            dsa.mla_decode(**{**dict(q=q, kv_cache=kv, indices=idx, sm_scale=0.1, seq_lens=sl), **bad})
    for bad in (dict(kv=host(kv)), dict(out=torch.zeros((2, 16, 512), dtype=torch.bfloat16)), dict(lse=torch.zeros((2, 16)))):
        with pytest.raises(ValueError):
            dsa.mla_prefill(**{**dict(q=q[:, 0], kv=kv, indices=idx[:, 0], sm_scale=0.1), **bad})
    assert not lib.launches
