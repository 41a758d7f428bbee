"""CPU-side checks of the scratch that calls share and of the 8-bit cache's limits."""

import ctypes
import os
import threading

import pytest
import torch

import _tak_b200 as T
import kv8_cache as C8

CPU = torch.device("cpu", 0)


def scratch(stream, nbytes):
    return T.workspace(CPU, ctypes.c_void_p(stream), nbytes)


def test_threads_on_one_stream_have_their_own_scratch(monkeypatch):
    """The launches of two threads' calls may alternate on a stream, so what one
    call hands from launch to launch must not lie in the other's buffer."""
    monkeypatch.setattr(T, "_ws", {})
    both, got = threading.Barrier(2), {}

    def work(name):
        both.wait()
        a = scratch(7, 64)
        both.wait()  # both threads are alive: neither has the other's identity
        b = scratch(7, 64)
        got[name] = (a.data_ptr(), b.data_ptr(), T.workspace_of(0, 7, 64).data_ptr(), scratch(8, 64).data_ptr())
        both.wait()

    threads = [threading.Thread(target=work, args=(n,)) for n in "ab"]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for first, again, by_index, other_stream in got.values():
        assert first == again == by_index and other_stream != first
    assert got["a"][0] != got["b"][0]


def test_scratch_grows_and_is_kept(monkeypatch):
    monkeypatch.setattr(T, "_ws", {})
    a = scratch(3, 64)
    assert scratch(3, a.numel()) is a
    b = scratch(3, a.numel() + 1)
    assert b.numel() > a.numel() and scratch(3, 64) is b and T.workspace_of(0, 3) is b


def test_scratch_of_ended_threads_is_given_back(monkeypatch):
    monkeypatch.setattr(T, "_ws", {})
    mine = scratch(3, 64)
    t = threading.Thread(target=scratch, args=(4, 64))
    t.start()
    t.join()
    assert len(T._ws) == 2
    scratch(5, 64)
    assert sorted(k[1] for k in T._ws) == [3, 5] and scratch(3, 64) is mine


def _cache(block, width):
    p = 4096  # never dereferenced: the sizes alone are looked at
    return C8._PACK.pack(p, 1, 1, 1, 1, p, 1, 1, 1, 1, p, 1, 1, 1, p, 1, 1, 1, p, 1, 1, 4, 2, block, 64, 16, 2, width, 0)


def test_rows_of_a_table_stay_below_the_reach_of_32_bits():
    """Kernels step past the last row in 32-bit positions: a table may not reach 2^31 - 2^16."""
    if not os.path.exists(T.LIB_PATH):
        pytest.skip("libtak_b200.so not built")
    size = T.lib().tak_kv8_attention_workspace_size
    for block in (16, 128, 65536):
        most = (2 ** 31 - 2 ** 16) // block
        assert size(_cache(block, most), 4, 1, 0, 1) >= 0  # accepted (these strides need no workspace)
        assert size(_cache(block, most + 1), 4, 1, 0, 1) == -1
        assert "max_blocks" in T.lib().tak_last_error().decode()


def test_workspace_size_of_refused_arguments():
    if not os.path.exists(T.LIB_PATH):
        pytest.skip("libtak_b200.so not built")
    size = T.lib().tak_kv8_attention_workspace_size
    assert size(_cache(16, 4), 4, 1, 64, 1) >= 0
    for bad in ((3, 1, 64, 1), (4, -1, 64, 1), (4, 65536, 64, 1), (4, 1, -1, 1), (4, 1, 2 ** 31, 1), (4, 1, 64, 3),
                (4, 1, 64, -1)):
        assert size(_cache(16, 4), *bad) == -1, bad
