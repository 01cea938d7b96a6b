"""What the paged operators pass to the library, on the CPU with a library that only records it."""
from __future__ import annotations

import struct

import pytest
import torch

from autosage_b200 import _native, paged

WORKSPACE = 35            # field of asg_paged_attention_args, counted in eights of bytes


class Recorder:
    """Stands in for the shared library."""

    def __init__(self):
        self.attention, self.written, self.sizes = [], [], []

    def asg_paged_attention(self, args):
        self.attention.append(struct.unpack("=38q", args))
        return 0

    def asg_paged_cache_write(self, args):
        self.written.append(struct.unpack("=31q", args))
        return 0

    def asg_paged_attention_workspace_bytes(self, n_heads, n_kv_heads, head_dim):
        self.sizes.append((torch.cuda.current_device(), n_heads, n_kv_heads, head_dim))
        return 4096 * (1 + torch.cuda.current_device())

    def asg_workspace_bytes(self, n_rows):
        return 4096


class Current:
    """Stands in for torch.cuda.device: two GPUs, the first of them current."""

    index, capturing = 0, set()

    def __init__(self, index):
        self.wanted = 0 if index is None else index

    def __enter__(self):
        self.before, Current.index = Current.index, self.wanted

    def __exit__(self, *_):
        Current.index = self.before


@pytest.fixture
def recorder(monkeypatch):
    library = Recorder()
    monkeypatch.setattr(_native, "_LIB", library)
    monkeypatch.setattr(_native, "_SCRATCH", {})
    monkeypatch.setattr(torch.cuda, "device", Current)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: Current.index)
    monkeypatch.setattr(_native, "_current_device", lambda: Current.index)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: Current.index in Current.capturing)
    monkeypatch.setattr(Current, "capturing", set())
    monkeypatch.setattr(_native, "_raw_stream", lambda index: 7)
    _native._paged_attention_bytes.cache_clear()
    yield library
    _native._paged_attention_bytes.cache_clear()


def attend():
    """One call below the checks of arguments."""
    pages, query = torch.zeros(3, 4, 2, 8), torch.zeros(2, 4, 8)
    crow, col, lengths = torch.tensor([0, 1, 3]), torch.tensor([2, 0, 1]), torch.tensor([3, 5])
    _native.paged_attention(crow, col, lengths, query, torch.empty_like(query), None, pages, pages.clone(), None, None, 1.0, 0)


def test_the_attention_has_a_workspace_of_its_own(recorder):
    """Another operator's launches, by another host thread on the same stream, may lie between the two of a call."""
    def other():
        return _native._scratch_on(torch.device("cpu"), None, 7, 4096)

    shared = other()
    attend()
    assert recorder.attention[0][WORKSPACE] != shared.data_ptr()
    attend()
    assert recorder.attention[1][WORKSPACE] == recorder.attention[0][WORKSPACE]     # kept between calls
    assert other().data_ptr() == shared.data_ptr()


def on_gpu(index):
    """The arguments of a call whose tensors say that they lie on GPU `index`."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        pages = [torch.zeros(3, 4, 2, 8, device=f"cuda:{index}") for _ in range(2)]
        crow, col, lengths = (torch.zeros(n, dtype=torch.long, device=f"cuda:{index}") for n in (3, 3, 2))
        query, out = (torch.zeros(2, 4, 8, device=f"cuda:{index}") for _ in range(2))
    return crow, col, lengths, query, out, None, *pages, None, None, 1.0, 0


@pytest.mark.filterwarnings("ignore:Accessing the data pointer")
def test_the_workspace_is_sized_for_the_gpu_of_the_tensors(recorder, monkeypatch):
    """Not for the current one, nor for the one that the first call went to."""
    asked = []

    def scratch_on(device, index, stream, need, *owner):
        asked.append((index, need))
        return torch.zeros(8192, dtype=torch.uint8)

    monkeypatch.setattr(_native, "_scratch_on", scratch_on)
    for index in (0, 1, 0, 1):
        _native.paged_attention(*on_gpu(index))
    assert asked == [(0, 4096), (1, 8192), (0, 4096), (1, 8192)] and Current.index == 0
    assert recorder.sizes == [(0, 4, 2, 8), (1, 4, 2, 8)]           # asked of the library once a GPU


def test_capture_is_asked_of_the_gpu_that_is_launched_on(recorder):
    Current.capturing.add(1)
    kept = _native._scratch_on(torch.device("cpu"), 0, 7, 100, "paged_attention")
    assert _native._scratch_on(torch.device("cpu"), 0, 7, 100, "paged_attention") is kept
    # what is captured on the other GPU comes from the graph's pool, whatever GPU is current
    first, second = (_native._scratch_on(torch.device("cpu"), 1, 7, 100, "paged_attention") for _ in range(2))
    assert first is not second and list(_native._SCRATCH) == [(0, 7, "paged_attention")]


def test_fake_tensors_are_refused_and_leave_no_workspace(recorder):
    """A fake tensor's address is 0; a workspace allocated among them would be fake too and serve the calls after it."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        pages = [torch.zeros(3, 4, 2, 8, device="cuda") for _ in range(2)]
        crow, col, lengths = (torch.zeros(n, dtype=torch.long, device="cuda") for n in (3, 3, 2))
        rows = torch.zeros(2, 2, 8, device="cuda")
        for call in (lambda: paged.csr_paged_attention(crow, col, lengths, rows, *pages),
                     lambda: paged.paged_cache_write(lengths, rows, rows, *pages),
                     lambda: paged.paged_cache_read(lengths, *pages)):
            with pytest.raises(RuntimeError, match="not fake ones"):
                call()
    assert recorder.attention == recorder.written == [] and _native._SCRATCH == {}


@pytest.mark.parametrize("made_in_inference", [(0,), (1,), (2,), (3,), (0, 2), (1, 3), (0, 1, 2, 3), ()], ids=str)
@pytest.mark.parametrize("later", [False, True], ids=["outside", "in inference mode"])
def test_a_write_counts_on_each_tensor_that_counts(recorder, monkeypatch, made_in_inference, later):
    """Tensors made in inference mode and others may be mixed: the write is made, and the others' versions rise."""
    monkeypatch.setattr(paged, "_require_native", lambda *_: None)
    monkeypatch.setattr(_native, "_page_pools", lambda *_: (0,) * 16)
    tensors = []
    for i, make in enumerate([lambda: torch.zeros(3, 4, 2, 8, dtype=torch.int8)] * 2 + [lambda: torch.zeros(3, 2, 4)] * 2):
        with torch.inference_mode(i in made_in_inference):
            tensors.append(make())
    before = {i: t._version for i, t in enumerate(tensors) if i not in made_in_inference}
    rows = torch.zeros(2, 2, 8)
    with torch.inference_mode(later):
        paged.paged_cache_write(torch.tensor([1, 2]), rows, rows, *tensors[:2], key_scales=tensors[2], value_scales=tensors[3])
    assert len(recorder.written) == 1
    assert all(tensors[i]._version == version + 1 for i, version in before.items())


def test_keys_and_values_are_not_written_to_the_same_memory(native_library):
    """The library says so before any CUDA call."""
    lib = _native.bind(str(native_library))

    def write(key=256, value=512, key_pages=1024, value_pages=2048, key_scales=0, value_scales=0, cache=0, n_tokens=2):
        pools = (key_pages, key_scales, 64, 16, 8, 0, 0, 0, value_pages, value_scales, 64, 16, 8, 0, 0, 0)
        code = lib.asg_paged_cache_write(_native._CACHE_ARGS.pack(128, n_tokens, key, 16, 8, value, 16, 8, *pools, 3, 4, 2, 8, 0, cache, 0))
        return code == -1 and b"to the same pages or scales" in lib.asg_last_error_string()

    assert write(value_pages=1024)
    assert write(cache=4, key_scales=4096, value_scales=4096)
    assert write(cache=4, key_scales=4096, value_scales=8192, value_pages=1024)
    assert not write(value_pages=1024, n_tokens=0)
    if not torch.cuda.is_available():                      # (with a GPU these would be launched)
        assert not write() and not write(value=256, value_pages=1024)
