"""The paged cache's structs as the library, the ctypes binding and the Rust
binding lay them out, and the page arithmetic of the kernels."""
import ctypes as C

import pytest

import obsmoe
import test_abi
from test_abi import header_struct_fields, rust_struct_layout


def test_paged_struct_layout_of_library_ctypes_and_rust_agree(monkeypatch):
    monkeypatch.setitem(test_abi.RUST_TYPES, "i64", (8, 8))
    v = obsmoe.paged_struct_layout()
    assert len(v) == 21
    at = 0
    for name, ct, rust in (("obs_paged_config", obsmoe.PagedConfig, "ObsPagedConfig"),
                           ("obs_paged_kv", obsmoe.PagedView, "ObsPagedKv")):
        fields = [f for f, _ in ct._fields_]
        assert [f for f in header_struct_fields(name) if f not in ("k", "v")] == [f for f in fields if f not in ("k", "v")]
        lib = (v[at], list(zip(fields, v[at + 1:at + 1 + len(fields)])))
        assert (C.sizeof(ct), [(f, getattr(ct, f).offset) for f in fields]) == lib
        assert rust_struct_layout(rust) == lib
        at += 1 + len(fields)


def test_null_arguments_are_errors_without_a_gpu():
    lib = obsmoe.lib()
    assert lib.obs_paged_init(None, None) == 1
    assert lib.obs_paged_append(None, None, None, None, 0, None, None, 1, None) == 1
    assert lib.obs_paged_decode(None, None, None, 0, None, 0, 0, 0.0, None, 0, None) == 1
    assert lib.obs_paged_prefill(None, None, None, 0, None, None, 1, 0, 0, 0.0, None) == 1
    assert lib.obs_paged_evict(None, None, None, None, None, 0, 1, 0, 0, None, None, None) == 1
    assert lib.obs_paged_attn_forward(None, 0, None, None, None, 1, None, None, None, None, 0, 0, None, 0, None) == 1


@pytest.mark.parametrize("page", [1, 2, 3, 5, 16, 63, 64, 100, 127, 128, 1000, 1023, 1024])
def test_page_of_a_position(page):
    """page = floor(j * (floor(2^32 / p) + 1) / 2^32), as the kernels have it, is j // p for every position of the
    longest sequence and a tile past it."""
    import numpy as np

    j = np.arange((1 << 20) + 256, dtype=np.uint64)
    magic = 0 if page == 1 else (1 << 32) // page + 1
    got = (j * np.uint64(magic)) >> np.uint64(32) if magic else j
    assert np.array_equal(got, j // np.uint64(page))
