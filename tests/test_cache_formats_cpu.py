"""Two instances whose pools are of different kinds (plain, e4m3) must not be bound to each other: host logic, no GPU."""
import json

import pytest
import torch

from distserve_amd import CacheConfig, ModelConfig, ParallelConfig, Worker, cabi

MODEL = ModelConfig.from_kv_shape(2, 8, 64, 4)


def a_worker(cache_dtype):
    """A worker's host side only: what binding looks at."""
    worker = object.__new__(Worker)
    worker.model_config, worker.parallel_config = MODEL, ParallelConfig()
    worker.cache_config = CacheConfig(16, 64, cache_dtype=cache_dtype)
    return worker


def handles(marks):
    """[pp][tp] = (k, v) of one stage whose ranks have these marks behind their words; no memory behind them."""
    words = [0] * cabi.KVM_HANDLE_WORDS
    return json.loads(json.dumps([[(words + m, words + m) for m in marks]]))       # they cross processes as plain data


PLAIN, CODED = [], [cabi.KVM_CACHE_E4M3]


@pytest.mark.parametrize("ours,theirs", [("auto", [CODED]), ("e4m3", [PLAIN]), ("auto", [PLAIN, CODED]),
                                         ("e4m3", [CODED, PLAIN]), ("e4m3", [[7]]), ("auto", [[1, 0]])])
def test_pools_of_another_kind_are_refused_before_any_is_bound(ours, theirs, monkeypatch):
    bound = []
    monkeypatch.setattr(torch.ops.block_migration_ops, "register_ipc_mem_handle_from", lambda *a: bound.append(a), raising=False)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda: None)
    with pytest.raises(RuntimeError, match="same cache_dtype"):
        a_worker(ours).register_kvcache_mem_handles(ParallelConfig(len(theirs)), handles(theirs))
    assert not bound


@pytest.mark.parametrize("ours,mark", [("auto", PLAIN), ("e4m3", CODED)])
def test_pools_of_the_same_kind_are_bound_without_their_mark(ours, mark, monkeypatch):
    bound = []
    monkeypatch.setattr(torch.ops.block_migration_ops, "register_ipc_mem_handle_from", lambda *a: bound.append(a), raising=False)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda: None)
    a_worker(ours).register_kvcache_mem_handles(ParallelConfig(2), handles([mark, mark]))
    assert len(bound) == 2 and all(len(a[1]) == len(a[2]) == cabi.KVM_HANDLE_WORDS for a in bound)


def test_the_op_takes_a_marked_handle_and_no_other_length():
    words, op = [0] * cabi.KVM_HANDLE_WORDS, torch.ops.block_migration_ops.register_ipc_mem_handle
    for k, v in ((words[1:], words), (words + [1], words), (words + [1, 1], words + [1, 1])):
        with pytest.raises(RuntimeError, match="words"):
            op(k, v, 2, 4, [1, 0, 1, 0], [1, 0, 1, 0])
    with pytest.raises(RuntimeError, match="kvmove error"):        # the words themselves are nobody's handle
        op(words + [1], words + [1], 2, 4, [1, 0, 1, 0], [1, 0, 1, 0])
