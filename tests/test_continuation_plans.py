"""How attention over paged caches is planned on the host, without a GPU: what a call asks of its scratch says how its keys are cut."""
from __future__ import annotations

import ctypes

import pytest

from holon_amd.kernels import build
from holon_amd.kernels.continuation import _ATTENTION, SYMBOLS


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(str(build.find_library() or build.build()))
    for name, (args, result) in SYMBOLS.items():
        getattr(lib, name).argtypes, getattr(lib, name).restype = args, result
    return lib


def _room(lib, heads, kv, dim, *, decode=(0, 0), chunk=(0, 0, 0), group=(0, 0, 0), tokens=None, q8=True, f32=False, page=16, window=0):
    """Bytes of scratch: decode (rows, longest), chunk (rows, most queries, longest), group (groups, most queries, longest prefix)."""
    rows = decode[0] + chunk[0]
    tokens = decode[0] + chunk[0] * chunk[1] if tokens is None else tokens
    return lib.holon_cache_attention_room(_ATTENTION.pack(
        0, int(q8), 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, tokens, 9, 9, 9, rows, *decode, *chunk, *group, heads, kv, dim, page, window, 0 if f32 else 1, 1.0))


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize(("heads", "kv", "dim"), [(65, 1, 64), (71, 1, 64), (128, 1, 64), (128, 1, 128), (66, 1, 256), (130, 2, 128)])
def test_heads_that_go_to_the_kernel_of_many_columns_are_not_cut_by_lengths(lib, heads, kv, dim, q8):
    """More than 64 heads on one: every row is cut into the same number of shares (at most 32), and the scratch holds their sums
    (dim numbers, a maximum and a sum each) and no list of the rows' own shares, which that kernel does not write."""
    for rows in (2, 3, 7, 33, 64):
        for longest in (4096, 4097, 8192, 100000):
            share = rows * heads * (dim + 2) * 4
            room = _room(lib, heads, kv, dim, decode=(rows, longest), q8=q8)
            assert room % share < 16 and room // share <= 32, (rows, longest, room)       # (whole pieces of 16 bytes)


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("q8", [True, False])
def test_every_bound_has_a_plan(lib, q8, f32):
    """Bounds that the entry point takes: no rows, rows of no key, groups of no key or no query, and more than there is."""
    if f32 and not q8:
        return
    for heads, kv, dim in ((1, 1, 64), (8, 2, 128), (20, 1, 256), (71, 1, 64)):
        for decode in ((0, 0), (1, 0), (2, 0), (40, 0), (3, 1), (1, 1 << 30)):
            for chunk in ((0, 0, 0), (1, 1, 0), (2, 2, 0), (3, 500, 1 << 30)):
                for group in ((0, 0, 0), (1, 0, 0), (1, 2, 0), (1, 0, 16), (1, 2, 16), (2, 600, 1 << 30)):
                    assert _room(lib, heads, kv, dim, decode=decode, chunk=chunk, group=group, q8=q8, f32=f32) >= 0


def test_scratch_is_in_whole_pieces_of_16_bytes(lib):
    """Partial sums are vectors of 16 bytes: those of a step's further kinds of rows begin behind the others', on a border."""
    rooms = set()
    for heads, kv, dim in ((1, 1, 64), (5, 1, 64), (3, 3, 128), (7, 1, 256)):
        for rows in (1, 3, 5):
            for longest in (5000, 7000, 9000, 30000):
                rooms |= {_room(lib, heads, kv, dim, decode=(rows, longest), q8=q8, f32=f32) for q8, f32 in ((True, False), (False, False), (True, True))}
                rooms |= {_room(lib, heads, kv, dim, decode=(rows, longest), chunk=(rows, most, longest)) for most in (3, 5, 400)}
                rooms.add(_room(lib, heads, kv, dim, decode=(rows, longest), group=(1, rows, longest)))
    assert len(rooms) > 50 and all(room % 16 == 0 for room in rooms)
