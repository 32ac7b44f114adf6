"""The work list of the many-tensor kernels (src/core/tensor_table.h) on the
CPU: every element is covered once, in launches that fit."""
import ctypes as C
import random

import pytest

CHUNK = 2048


def pack(core, sizes, room, chunk=CHUNK):
    L = core.lib()
    L.nb_pack_tensors.argtypes = [C.c_void_p, C.c_size_t, C.c_int, C.c_uint, C.c_int, C.c_void_p, C.c_void_p, C.c_void_p]
    n = len(sizes)
    arr = (C.c_uint64 * n)(*sizes)
    out = []
    for k in range(L.nb_pack_tensors(arr, n, room, chunk, -1, None, None, None)):
        tensor, first, chunks = (C.c_int * n)(), (C.c_uint * n)(), C.c_uint()
        m = L.nb_pack_tensors(arr, n, room, chunk, k, tensor, first, C.byref(chunks))
        out.append((list(tensor)[:m], list(first)[:m], chunks.value))
    return out


@pytest.mark.parametrize("chunk", [2048, 8192])
@pytest.mark.parametrize("room", [1, 2, 7, 400])
def test_every_chunk_finds_its_tensor(core, room, chunk):
    rng = random.Random(room)
    sizes = [rng.choice([0, 1, 2047, 2048, 2049, 8192, 8193, rng.randrange(1, 50000)]) for _ in range(60)]
    L = core.lib()
    L.nb_find_tensor.argtypes = [C.c_uint, C.c_void_p, C.c_int]
    covered = {}
    for tensor, first, chunks in pack(core, sizes, room, chunk):
        assert 1 <= len(tensor) <= room and first[0] == 0
        arr = (C.c_uint * len(first))(*first)
        for c in range(chunks):
            i = L.nb_find_tensor(c, arr, len(first))
            assert first[i] <= c and (i + 1 == len(first) or c < first[i + 1])
            begin = (c - first[i]) * chunk
            assert begin < sizes[tensor[i]]
            covered.setdefault(tensor[i], []).append(begin)
    for i, n in enumerate(sizes):
        assert sorted(covered.get(i, [])) == list(range(0, n, chunk))


def test_empty_and_huge_lists(core):
    assert pack(core, [0, 0], 4) == []
    # Offsets of a tensor beyond 2^32 elements are counted in 64 bits; more than
    # 2^31 chunks in one launch are split, and in one tensor refused.
    big = (1 << 33) + 1
    assert pack(core, [big], 4)[0][2] == (1 << 22) + 1
    assert len(pack(core, [((1 << 31) - 2) * CHUNK, CHUNK, CHUNK], 4)) == 2
    assert pack(core, [(1 << 31) * CHUNK], 4) == []
