"""What PagedKVCache does on the host: which calls it takes in which state, and what becomes of its pages.  The kernels are
replaced by recorders, so no device is needed."""
import pytest
import torch

from swiftlm_b200 import kernels
from swiftlm_b200.kv_cache import PagedKVCache


@pytest.fixture
def cache(monkeypatch):
    """Two sequences, pages of 4 tokens, on the CPU; kv_append and kv_commit move the lengths and nothing else."""
    calls = []

    def append(k_new, v_new, k_cache, v_cache, kv_len=None, len_all=0, page_table=None, kv_len_out=None):
        kv_len_out.copy_(kv_len + k_new.shape[2])

    def commit(kv_len, count, block=16):
        kv_len += count.clamp(0, block)

    monkeypatch.setattr(kernels, "kv_append", append)
    monkeypatch.setattr(kernels, "kv_commit", commit)
    for name in ("decode_sdpa", "prompt_sdpa", "attention_mass", "kv_evict"):
        monkeypatch.setattr(kernels, name, lambda *a, _name=name, **k: calls.append((_name, k)))
    c = PagedKVCache(2, 1, 8, 4, num_pages=16, max_pages=8, device="cpu", track_mass=True)
    c.calls = calls
    return c


def rows(T):
    return torch.zeros(2, 1, T, 8, dtype=torch.bfloat16)


def test_attention_over_the_committed_tokens_is_refused_between_append_and_commit(cache):
    q, lse = torch.zeros(2, 1, 3, 8, dtype=torch.bfloat16), torch.zeros(2, 1, 3)
    cache.extend(rows(6), rows(6), [6, 5])
    cache.attend_prompt(q, 1.0)
    cache.add_mass(q, lse, 1.0)
    assert [c[0] for c in cache.calls] == ["prompt_sdpa", "attention_mass"]
    cache.append_block(rows(3), rows(3))
    with pytest.raises(RuntimeError):
        cache.attend_prompt(q, 1.0)                 # its rows would be taken for tokens 3 .. 5 in place of 6 .. 8
    with pytest.raises(RuntimeError):
        cache.add_mass(q, lse, 1.0)
    assert len(cache.calls) == 2
    cache.commit(torch.tensor([3, 1], dtype=torch.int32))
    cache.attend_prompt(q, 1.0)
    cache.add_mass(q, lse, 1.0)
    assert [c[0] for c in cache.calls] == ["prompt_sdpa", "attention_mass"] * 2


def test_sync_between_append_and_commit_keeps_the_pages_of_the_block(cache):
    cache.extend(rows(4), rows(4), [4, 3])
    cache.extend(rows(4), rows(4), [2, 1])          # upper bounds 8 and 8, committed 6 and 4
    cache.append_block(rows(3), rows(3))            # rows 6 .. 8 and 4 .. 6: three and two pages
    before = [cache.pages_of(b) for b in range(2)]
    assert cache.sync().tolist() == [6, 4]
    assert cache.pages_of(0) == before[0][:3] and cache.pages_of(1) == before[1][:2]
    for b, n in enumerate((3, 2)):
        assert cache.page_table[b, :n].tolist() == before[b][:n] and (cache.page_table[b, n:] == -1).all()
    cache.commit(torch.tensor([3, 3], dtype=torch.int32))
    assert cache.sync().tolist() == [9, 7]
    assert len(cache.pages_of(0)) == 3 and len(cache.pages_of(1)) == 2
