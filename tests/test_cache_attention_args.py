"""Refusals of the cache operators, without a device: every argument is checked before the GPU is touched."""
import pytest

from swiftlm_b200 import _lib

FAKE = 0x1000   # never dereferenced


def call(op, **over):
    L = _lib.lib()
    a = dict(q=FAKE, k=FAKE, v=FAKE, page_table=None, q_len=None, kv_len=None, out=FAKE, lse=None, mass=None, ws=None, ws_bytes=0, B=1, Hq=16,
             Hkv=2, T=32, D=256, N=64, page_tokens=0, max_pages=0, num_pages=0, mass_stride=0, window=0, sinks=0, scale=0.0625,
             dtype=_lib.BF16, kv_len_out=FAKE, mass_out=FAKE, kept=FAKE, budget=8, recent=2)
    a.update(over)
    if op == "decode":
        return L.dflash_decode_sdpa(*(a[n] for n in "q k v page_table kv_len out lse mass ws ws_bytes B Hq Hkv D N page_tokens max_pages num_pages "
                                      "mass_stride window sinks scale dtype".split()), None)
    if op == "prompt":
        return L.dflash_prompt_sdpa(*(a[n] for n in "q k v page_table q_len kv_len out lse ws ws_bytes B Hq Hkv T D N page_tokens max_pages "
                                      "num_pages window sinks scale dtype".split()), None)
    if op == "mass":
        a = dict(a, lse=over.get("lse", FAKE), mass=over.get("mass", FAKE), mass_stride=over.get("mass_stride", a["N"]))
        return L.dflash_attention_mass(*(a[n] for n in "q k page_table q_len kv_len lse mass ws ws_bytes B Hq Hkv T D N page_tokens max_pages "
                                         "num_pages mass_stride window sinks scale dtype".split()), None)
    a = dict(a, mass=over.get("mass", FAKE), kv_len=over.get("kv_len", FAKE), mass_stride=over.get("mass_stride", a["N"]))
    return L.dflash_kv_evict(*(a[n] for n in "k v page_table kv_len mass kv_len_out mass_out kept ws ws_bytes B Hkv D N page_tokens max_pages "
                               "num_pages mass_stride budget recent sinks dtype".split()), None)


@pytest.mark.parametrize("op", ["decode", "prompt", "mass"])
def test_attention_refusals(op):
    bad, un = _lib.ERR_INVALID_ARG, _lib.ERR_UNSUPPORTED
    assert call(op, q=None) == bad and call(op, k=None) == bad
    assert call(op, B=0) == bad and call(op, N=0) == bad and call(op, Hkv=-2) == bad
    assert call(op, dtype=_lib.F32) == un and call(op, dtype=9) == un
    assert call(op, D=96) == un and call(op, D=512) == un
    assert call(op, Hq=15) == un
    assert call(op, window=-1) == bad and call(op, sinks=-1) == bad
    assert call(op, scale=float("nan")) == bad and call(op, scale=float("inf")) == bad
    assert call(op, scale=0.0) == bad and call(op, scale=-0.1) == bad and call(op, scale=1e-38) == bad
    assert call(op, q=FAKE + 8) == bad and call(op, k=FAKE + 2) == bad
    assert call(op, page_table=FAKE, page_tokens=24, max_pages=9, num_pages=9) == un
    assert call(op, page_table=FAKE, page_tokens=16, max_pages=3, num_pages=9) == bad      # 48 < N
    assert call(op, page_table=FAKE, page_tokens=16, max_pages=4, num_pages=0) == bad
    if op != "decode":
        assert call(op, T=0) == bad
    if op == "mass":
        assert call(op, lse=None) == bad and call(op, mass=None) == bad and call(op, mass_stride=63) == bad
    else:
        assert call(op, out=None) == bad and call(op, v=None) == bad
    if op == "decode":
        assert call(op, mass=FAKE, mass_stride=63) == bad


def test_workspace_is_checked():
    L = _lib.lib()
    need = L.dflash_decode_sdpa_workspace_bytes(4, 16, 2, 256, 100000, 0, 0, 1)
    assert need > 0
    assert call("decode", B=4, N=100000, mass=FAKE, mass_stride=100000, ws=FAKE, ws_bytes=need - 1) == _lib.ERR_WORKSPACE
    assert call("decode", B=4, N=100000, mass=FAKE, mass_stride=100000) == _lib.ERR_WORKSPACE
    assert call("evict", kept=None) == _lib.ERR_WORKSPACE
    assert L.dflash_kv_evict_workspace_bytes(1, 2, 64, 8) >= 2 * 8 * 4
    # sizes of calls that cannot be made are 0
    assert L.dflash_decode_sdpa_workspace_bytes(0, 16, 2, 256, 100, 0, 0, 1) == 0
    assert L.dflash_prompt_sdpa_workspace_bytes(1, 15, 2, 8, 256, 100) == 0
    assert L.dflash_attention_mass_workspace_bytes(1, 16, 2, 0, 256, 100) == 0
    assert L.dflash_kv_evict_workspace_bytes(1, 2, 64, 0) == 0


def test_evict_refusals():
    bad, un = _lib.ERR_INVALID_ARG, _lib.ERR_UNSUPPORTED
    for name in ("k", "v", "mass", "kv_len", "kv_len_out", "mass_out"):
        assert call("evict", **{name: None}) == bad, name
    assert call("evict", budget=0) == bad and call("evict", recent=-1) == bad and call("evict", sinks=-1) == bad
    assert call("evict", recent=5, sinks=4) == bad                                          # 9 > 8
    assert call("evict", recent=2 ** 31 - 1, sinks=2 ** 31 - 1) == bad
    assert call("evict", dtype=_lib.U8) == un
    assert call("evict", D=4) == bad and call("evict", k=FAKE + 4) == bad
    assert call("evict", mass_stride=63) == bad
    assert call("evict", page_table=FAKE, page_tokens=16, max_pages=3, num_pages=9) == bad


def test_python_side_refuses_cpu_tensors():
    import torch

    from swiftlm_b200 import kernels
    q, k = torch.zeros(1, 4, 64), torch.zeros(1, 2, 8, 64)
    with pytest.raises(RuntimeError):
        kernels.decode_sdpa(q, k, k, 1.0)
    with pytest.raises(RuntimeError):
        kernels.prompt_sdpa(q[:, :, None], k, k, 1.0)
    with pytest.raises(RuntimeError):
        kernels.attention_mass(q[:, :, None], k, torch.zeros(1, 4, 1), 1.0, torch.zeros(1, 2, 8))
    with pytest.raises(RuntimeError):
        kernels.kv_evict(k, k, torch.zeros(1, 2, 8), torch.zeros(1, dtype=torch.int32), 4, 1)


@pytest.mark.parametrize("op", ["decode", "prompt", "mass", "evict"])
def test_lengths_whose_positions_pass_32_bits_are_refused(op):
    for n in (2 ** 29 + 1, 2 ** 31 - 1):
        assert call(op, N=n, mass_stride=n) == _lib.ERR_UNSUPPORTED
        if op in ("prompt", "mass"):
            assert call(op, T=n) == _lib.ERR_UNSUPPORTED
    L, n = _lib.lib(), 2 ** 31 - 1
    assert L.dflash_decode_sdpa_workspace_bytes(1, 16, 2, 256, n, 0, 0, 1) == 0
    assert L.dflash_prompt_sdpa_workspace_bytes(1, 16, 2, 8, 256, n) == 0 and L.dflash_prompt_sdpa_workspace_bytes(1, 16, 2, n, 256, 8) == 0
    assert L.dflash_attention_mass_workspace_bytes(1, 16, 2, 8, 256, n) == 0 and L.dflash_attention_mass_workspace_bytes(1, 16, 2, n, 256, 8) == 0
    assert L.dflash_kv_evict_workspace_bytes(1, 2, n, 8) == 0
