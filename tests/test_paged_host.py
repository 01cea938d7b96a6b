"""The paged cache's checks of arguments, on the CPU, and the float64 rounding that its GPU tests compare with."""
from __future__ import annotations

import pytest
import torch

from autosage_b200 import paged
from paged_reference import LARGEST, e4m3_values, nearest_code_value, quantise


def pages(kind=torch.float32, n=3, page=4, heads=2, dim=8):
    return torch.zeros(n, page, heads, dim).to(kind)


def scales(n=3, page=4, heads=2):
    return torch.zeros(n, heads, page)


def table():
    return torch.tensor([0, 1, 3]), torch.tensor([2, 0, 1]), torch.tensor([3, 5])


def test_alias_package_has_the_module():
    import autosage

    from autosage.paged import csr_paged_attention

    assert csr_paged_attention is paged.csr_paged_attention and autosage.paged is paged


def attend(**change):
    crow, col, lengths = table()
    call = dict(crow=crow, col=col, lengths=lengths, query=torch.zeros(2, 4, 8), key_pages=pages(), value_pages=pages())
    call.update(change)
    return paged.csr_paged_attention(**call)


@pytest.mark.parametrize("change, error, message", [
    (dict(crow=torch.tensor([0.0, 1, 3])), TypeError, "crow must use integer"),
    (dict(crow=torch.tensor([0, 3])), ValueError, "crow must contain"),
    (dict(crow=torch.tensor([[0, 1, 3]])), ValueError, "crow must be one-dimensional"),
    (dict(lengths=torch.tensor([3])), ValueError, "lengths must contain"),
    (dict(query=torch.zeros(2, 3, 8)), ValueError, "multiple of n_kv_heads"),
    (dict(query=torch.zeros(2, 0, 8)), ValueError, "multiple of n_kv_heads"),
    (dict(query=torch.zeros(2, 4, 7)), ValueError, "head_dim"),
    (dict(query=torch.zeros(2, 32)), ValueError, "query must have shape"),
    (dict(query=torch.zeros(2, 4, 8).double()), TypeError, "query must be float32"),
    (dict(query=torch.zeros(2, 4, 8).half()), TypeError, "type of the query"),
    (dict(value_pages=pages(page=5)), ValueError, "same \\[n_pages"),
    (dict(value_pages=pages(torch.bfloat16)), TypeError, "pages must both"),
    (dict(key_pages=pages(torch.int32), value_pages=pages(torch.int32)), TypeError, "pages must both"),
    (dict(key_pages=pages(dim=264), value_pages=pages(dim=264)), ValueError, "at most 256"),
    (dict(key_pages=pages(torch.int8), value_pages=pages(torch.int8)), ValueError, "need key_scales"),
    (dict(key_pages=pages(torch.int8), value_pages=pages(torch.int8), key_scales=scales()), ValueError, "need value_scales"),
    (dict(key_pages=pages(torch.int8), value_pages=pages(torch.int8), key_scales=scales().half(), value_scales=scales()),
     TypeError, "key_scales must be float32"),
    (dict(key_pages=pages(torch.int8), value_pages=pages(torch.int8), key_scales=scales(), value_scales=scales(page=5)),
     ValueError, "value_scales must have shape"),
    (dict(key_scales=scales(), value_scales=scales()), ValueError, "8-bit pages only"),
    (dict(key_pages=pages(dim=16)[..., ::2]), ValueError, "contiguous"),
    (dict(window=0), ValueError, "window must be positive"),
    (dict(window=1.5), TypeError, "whole number"),
    (dict(), RuntimeError, "needs CUDA"),
])
def test_attention_refuses(change, error, message):
    with pytest.raises(error, match=message):
        attend(**change)


def write(**change):
    call = dict(slots=torch.tensor([0, 5, -1]), key=torch.zeros(3, 2, 8), value=torch.zeros(3, 2, 8), key_pages=pages(),
                value_pages=pages())
    call.update(change)
    return paged.paged_cache_write(**call)


@pytest.mark.parametrize("change, error, message", [
    (dict(slots=torch.tensor([0, 5])), ValueError, "one slot per token"),
    (dict(slots=torch.tensor([0.0, 5, 1])), TypeError, "slots must use integer"),
    (dict(key=torch.zeros(3, 2, 7)), ValueError, "same \\[tokens"),
    (dict(key=torch.zeros(3, 1, 8), value=torch.zeros(3, 1, 8)), ValueError, "same \\[tokens"),
    (dict(key=torch.zeros(3, 2, 8).half()), TypeError, "must both be"),
    (dict(key=torch.zeros(3, 2, 8).half(), value=torch.zeros(3, 2, 8).half()), TypeError, "type of key and value"),
    (dict(key_pages=torch.zeros(1, 4, 2, 8).expand(3, 4, 2, 8)), ValueError, "must not repeat memory"),
    (dict(), RuntimeError, "needs CUDA"),
])
def test_write_refuses(change, error, message):
    with pytest.raises(error, match=message):
        write(**change)


def test_read_refuses():
    slots = torch.tensor([0, 5])
    with pytest.raises(TypeError, match="dtype must be"):
        paged.paged_cache_read(slots, pages(), pages(), dtype=torch.int8)
    with pytest.raises(ValueError, match="one-dimensional"):
        paged.paged_cache_read(slots.view(1, 2), pages(), pages())
    with pytest.raises(RuntimeError, match="needs CUDA"):
        paged.paged_cache_read(slots, pages(), pages())


def test_library_checks_come_before_any_cuda_call(native_library):
    """Bad sizes given to the C entry points are reported on a host without a GPU."""
    from autosage_b200 import _native

    lib = _native.bind(str(native_library))

    def says(code, wanted, text):
        assert code == wanted and text in lib.asg_last_error_string(), lib.asg_last_error_string()

    def attention(n_rows=1, n_cols=0, n_pages=0, page=16, heads=4, kv=2, dim=64, window=0, kind=0, cache=0, data=0):
        pool = (data, 0, 0, 0, 0, 0, 0, 0)
        return lib.asg_paged_attention(_native._ATTENTION_ARGS.pack(
            0, 0, 0, n_rows, n_cols, 0, 0, 0, 0, 0, *pool, *pool, n_pages, page, heads, kv, dim, window, kind, cache, 1.0, 0, 0, 0))

    says(attention(dim=257), -4, b"256 features")
    says(attention(page=0), -1, b"page_size")
    says(attention(page=1 << 30), -4, b"index range")
    says(attention(heads=5), -1, b"multiple of n_kv_heads")
    says(attention(heads=1 << 40), -1, b"multiple of n_kv_heads")
    says(attention(kv=1 << 40, heads=1 << 40), -4, b"index range")
    says(attention(kind=3), -1, b"type of the tokens")
    says(attention(cache=9), -1, b"type of the pages")
    says(attention(cache=1), -1, b"8-bit type")
    says(attention(window=-1), -1, b"window")
    says(attention(n_cols=1 << 31), -4, b"n_cols")
    says(attention(n_pages=3), -1, b"pages must not be null")
    says(attention(n_pages=3, cache=4, data=256), -1, b"8-bit pages need scales")
    says(attention(), -1, b"must not be null")
    assert attention(n_rows=0) == 0

    def cache(entry, n_tokens=4, page=16, kind=0, cache=0, n_pages=0, data=0):
        pool = (data, 0, 0, 0, 0, 0, 0, 0)
        return entry(_native._CACHE_ARGS.pack(0, n_tokens, 0, 0, 0, 0, 0, 0, *pool, *pool, n_pages, page, 2, 64, kind, cache, 0))

    for entry in (lib.asg_paged_cache_write, lib.asg_paged_cache_read):
        says(cache(entry), -1, b"slots, key and value")
        says(cache(entry, n_tokens=-1), -1, b"n_tokens")
        says(cache(entry, kind=4), -1, b"type of the tokens")
        says(cache(entry, n_tokens=0, n_pages=1, cache=3, data=256), -1, b"8-bit pages need scales")
        says(entry(None), -1, b"args must not be null")
        assert cache(entry, n_tokens=0) == 0
    says(cache(lib.asg_paged_cache_write, n_tokens=0, cache=1), -1, b"8-bit type")
    says(lib.asg_paged_attention(None), -1, b"args must not be null")
    assert lib.asg_paged_attention_workspace_bytes(32, 8, 128) % 256 == 0
    assert lib.asg_paged_attention_workspace_bytes(32, 7, 128) == 0


def test_packed_arguments_have_the_layout_of_the_header(tmp_path):
    """The structs of the header have as many 8-byte fields as the binding packs."""
    import shutil
    import subprocess
    from pathlib import Path

    from autosage_b200 import _native

    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("no C compiler")
    source = tmp_path / "sizes.c"
    source.write_text('#include "autosage_b200.h"\n#include <stdio.h>\nint main(void) {'
                      ' printf("%zu %zu %zu", sizeof(asg_paged_cache_args), sizeof(asg_paged_attention_args),'
                      ' offsetof(asg_paged_attention_args, scale)); return 0; }')
    include = Path(_native.__file__).resolve().parent.parent / "include"
    subprocess.run([gcc, "-std=c99", "-Wall", "-Werror", f"-I{include}", str(source), "-o", str(tmp_path / "sizes")], check=True)
    sizes = subprocess.run([str(tmp_path / "sizes")], capture_output=True, text=True, check=True).stdout.split()
    assert [int(n) for n in sizes] == [_native._CACHE_ARGS.size, _native._ATTENTION_ARGS.size, 34 * 8]


@pytest.mark.parametrize("kind", list(LARGEST))
def test_reference_rounding_takes_the_nearest_code(kind):
    values = e4m3_values() if kind != torch.int8 else torch.arange(128).double()
    assert torch.equal(nearest_code_value(values, kind), values) and torch.equal(nearest_code_value(-values, kind), -values)
    middle = (values[1:] + values[:-1]) / 2
    even = values[1:].clone()
    even[::2] = values[:-1][::2]                                   # border i lies between codes i and i + 1
    assert torch.equal(nearest_code_value(middle, kind), even)
    assert torch.equal(nearest_code_value(middle * (1 - 2.0 ** -50), kind), values[:-1])
    assert torch.equal(nearest_code_value(middle * (1 + 2.0 ** -50), kind), values[1:])
    x = torch.tensor([[0.0, 0.0], [1.0, -2.0]]).double()
    code, scale = quantise(x, kind)
    assert code[0].abs().max() == 0 and scale[0] == 0 and code[1, 1] == -LARGEST[kind]
