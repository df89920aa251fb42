"""Steps of several new tokens per request, without a GPU: refusals of the entry points, and what the oracle says of requests that a
step cannot take."""
import ctypes as C

import pytest
import torch

from lsvd_b200 import ChunkState, LsvdError, _lib, chunk
from oracle import attention
from test_chunk_cpu import _chunk_args, _maps_args, lib      # noqa: F401  (a fixture)


def test_maps_tell_an_empty_free_list_from_a_missing_one(lib):      # noqa: F811
    """A list of no entries may have no address; then its head still has to be there, and its length is zero."""
    a = _maps_args()
    a.free_pages = None                                   # four entries, no address
    assert lib.lsvd_chunk_maps(C.byref(a), None) == _lib.ERR_INVALID_ARG
    a = _maps_args()
    a.free_pages, a.num_free, a.free_head_out = None, 0, None
    assert lib.lsvd_chunk_maps(C.byref(a), None) == _lib.ERR_INVALID_ARG


def test_attention_refuses_misaligned_slots(lib):      # noqa: F811
    a = _chunk_args()
    a.mem_index = 4097
    assert lib.lsvd_attn_chunk(C.byref(a), None) == _lib.ERR_INVALID_ARG


def test_maps_refuse_a_negative_bound(lib):      # noqa: F811
    a = _maps_args()
    a.max_new_in_batch = -1
    assert lib.lsvd_chunk_maps(C.byref(a), None) == _lib.ERR_INVALID_ARG


def test_oracle_maps_refuse_more_tokens_than_the_bound():
    table, r2t = [[0, -1], [1, -1]], [[-1] * 32 for _ in range(2)]
    start, seq, mem, pos, head, refused = attention.chunk_maps([0, 1], [3, 3], [5, 4], table, 16, r2t, 9, 64, [2, 3], 0, max_new=4)
    assert refused == [0] and seq == [3, 7] and start == [0, 5, 9] and mem == [-1] * 5 + [19, 20, 21, 22] and head == 0


def test_state_raises_what_was_reported_once(lib):      # noqa: F811
    st = ChunkState.paged(rows=2, max_len_in_batch=33, max_tokens=5, max_new_in_batch=3, num_pages=7, page_size=16, device="cpu")
    st.check()
    st.status_word.fill_(_lib.ERR_BOUNDS)
    with pytest.raises(LsvdError):
        st.check()
    st.check()


def test_kept_workspaces_of_two_devices(monkeypatch):
    """Steps that alternate between devices find their own again."""
    import contextlib
    monkeypatch.setattr(chunk, "attn_chunk_workspace_bytes", lambda state, layout, n: 1000 * n)
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    kept, cpu, meta = [], torch.device("cpu"), torch.device("meta")
    a, b = chunk.kept_workspace(kept, None, None, 2, cpu), chunk.kept_workspace(kept, None, None, 1, meta)
    for _ in range(3):
        assert chunk.kept_workspace(kept, None, None, 2, cpu) is a and chunk.kept_workspace(kept, None, None, 1, meta) is b
    big = chunk.kept_workspace(kept, None, None, 3, cpu)
    assert big.numel() == 4000 and [w.numel() for w in kept] == [2000, 1000, 4000]
    assert chunk.kept_workspace(kept, None, None, 1, cpu) is big and kept[0] is a


def test_status_words_have_to_be_where_the_kernels_run():
    gpu, cpu = torch.device("cuda", 0), torch.device("cpu")
    assert chunk._status(None, gpu) is None
    word = torch.zeros(1, dtype=torch.int32)
    assert chunk._status(word, cpu) == word.data_ptr()
    for bad, dev in ((word, gpu), (word.long(), cpu), (word[:0], cpu), (torch.zeros(1), cpu)):
        with pytest.raises(ValueError):
            chunk._status(bad, dev)


def test_bounds_are_held_not_wrapped():
    assert [chunk._bound(n) for n in (0, 5, -3, 2 ** 31 - 1, 2 ** 31, 2 ** 32 + 1)] == [0, 5, -3, 2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1]
