"""The cache operators where a row's softmax or a call's size leaves the ordinary path: queries that are no numbers, weights
far below the largest, tables and loops that only large batches reach.  Plain forms in 64 bits."""
import math

import pytest
import torch

from tests.test_gpu_cache_attention import K, Problem

pytestmark = pytest.mark.gpu
INF, NAN = math.inf, math.nan


# head dimension 64, 128, 256; one CTA for a unit, and units cut into pieces that are joined
@pytest.mark.parametrize("D,N,page", [(64, 70, 0), (128, 300, 16), (256, 300, 64), (256, 30000, 0)])
@pytest.mark.parametrize("value", [NAN, INF])
def test_decode_of_a_query_that_is_no_number(D, N, page, value):
    """Scores q.k of which one is NaN or +infinity have no softmax: out, lse and the weights of that head are NaN, and nothing of
    it reaches another head's output."""
    B, Hq, Hkv = 2, 6, 2
    x = Problem(B, Hq, Hkv, 1, D, N, "bf16", page, [N, max(1, N // 3)], seed=D + N)
    q = x.q[:, :, 0].clone()
    q[0, 1, 3] = value                                    # a head of KV head 0 of sequence 0
    cap = N if not page else x.table.shape[1] * page
    mass, clean_mass = (torch.full((B, Hkv, cap), 0.25, device="cuda") for _ in range(2))
    window = 40 if N < 1000 else 20000
    args = dict(kv_len=x.kv_len, page_table=x.table, window=window, sinks=3)
    clean, clean_lse = K().decode_sdpa(x.q[:, :, 0], x.k, x.v, x.scale, mass=clean_mass, return_lse=True, **args)
    got, lse = K().decode_sdpa(q, x.k, x.v, x.scale, mass=mass, return_lse=True, **args)
    K().device_status()
    hit = torch.zeros(B, Hq, dtype=torch.bool, device="cuda")
    hit[0, 1] = True
    assert torch.isnan(got[hit]).all() and torch.isnan(lse[hit]).all()
    assert torch.equal(got[~hit], clean[~hit]) and torch.equal(lse[~hit], clean_lse[~hit])
    n = torch.arange(cap, device="cuda")
    seen = (n < N) & ((n >= N - window) | (n < 3))
    assert torch.isnan(mass[0, 0, seen]).all()
    keep = torch.ones_like(mass, dtype=torch.bool)
    keep[0, 0] = ~seen
    assert torch.equal(mass[keep], clean_mass[keep])


@pytest.mark.parametrize("Hq,Hkv,T,D,N,page,window,sinks", [
    (4, 2, 70, 64, 90, 0, 0, 0),                           # whole units
    (6, 2, 40, 128, 300, 16, 30, 3),
    (4, 2, 130, 256, 300, 64, 0, 0),                       # a pair of CTAs
    (4, 1, 9, 256, 30000, 0, 0, 0),                        # units cut into pieces
    (4, 1, 9, 64, 30000, 0, 0, 0),
])
@pytest.mark.parametrize("value", [NAN, INF])
def test_prompt_row_that_is_no_number(Hq, Hkv, T, D, N, page, window, sinks, value):
    """out and lse of that row are NaN; every other row has the bits that it has without it."""
    B = 2
    x = Problem(B, Hq, Hkv, T, D, N, "bf16", page, [N, N - 5], seed=D + N)
    q = x.q.clone()
    rows = [(0, 1, T - 1), (1, Hq - 1, T // 2)]
    hit = torch.zeros(B, Hq, T, dtype=torch.bool, device="cuda")
    for b, h, t in rows:
        q[b, h, t, 5] = value
        hit[b, h, t] = True
    args = dict(kv_len=x.kv_len, page_table=x.table, window=window, sinks=sinks, return_lse=True)
    clean, clean_lse = K().prompt_sdpa(x.q, x.k, x.v, x.scale, **args)
    got, lse = K().prompt_sdpa(q, x.k, x.v, x.scale, **args)
    K().device_status()
    assert torch.isnan(got[hit]).all() and torch.isnan(lse[hit]).all()
    assert torch.equal(got[~hit], clean[~hit]) and torch.equal(lse[~hit], clean_lse[~hit])


@pytest.mark.parametrize("Hq,Hkv,T,D,N,page,window,sinks", [
    (4, 2, 70, 64, 90, 0, 0, 0),
    (6, 2, 40, 128, 300, 16, 30, 3),
    (3, 1, 16, 256, 700, 64, 0, 0),                        # 126 rows of a query tile in use
    (4, 1, 300, 128, 5000, 0, 0, 0),                       # several query tiles, units cut into pieces
    (160, 1, 5, 64, 400, 0, 100, 7),                       # two groups of heads
])
@pytest.mark.parametrize("case", ["lse", NAN, INF])
def test_mass_of_a_row_that_is_no_number(Hq, Hkv, T, D, N, page, window, sinks, case):
    """A log-sum-exp that is NaN (given as such, or that of a query with a NaN or an infinity) makes the masses of the tokens
    that the row sees NaN; all other masses have the bits that they have without it."""
    B = 2
    x = Problem(B, Hq, Hkv, T, D, N, "f16", page, [N, N - 5], seed=D + N)
    args = dict(kv_len=x.kv_len, page_table=x.table, window=window, sinks=sinks)
    lse = K().prompt_sdpa(x.q, x.k, x.v, x.scale, return_lse=True, **args)[1]
    cap = N if not page else x.table.shape[1] * page
    clean, mass = (torch.full((B, Hkv, cap), 0.5, device="cuda") for _ in range(2))
    K().attention_mass(x.q, x.k, lse, x.scale, clean, **args)
    q, bad_lse = x.q.clone(), lse.clone()
    hit = torch.zeros(B, Hkv, cap, dtype=torch.bool, device="cuda")
    for b, h, t in [(0, 1, T // 2), (1, Hq - 1, T - 2)]:
        if case == "lse":
            bad_lse[b, h, t] = NAN
        else:
            q[b, h, t, 5] = case
        hit[b, h // (Hq // Hkv), :x.kv[b]] |= x.seen(b, window, sinks)[t]
    if case != "lse":
        bad_lse = K().prompt_sdpa(q, x.k, x.v, x.scale, return_lse=True, **args)[1]
    K().attention_mass(q, x.k, bad_lse, x.scale, mass, **args)
    K().device_status()
    assert torch.isnan(mass[hit]).all()
    assert torch.equal(mass[~hit], clean[~hit])


def light_tokens(B, T, D, N, seed):
    """f16: token 0 takes nearly all of the weight and has no value; the others weigh 2^-26.5 of it each, all their values are in
    [1, 2].  (q, k, v, out in 64 bits, bound).  Bound: half a step u of the output, its subnormal half step 2^-25, half a step u of
    each weight and, for weights below the smallest normal one, half of 2^-24 at a lift of 2^7: 2^-32 each."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.zeros(B, 2, T, D, device="cuda", dtype=torch.float16)
    k, v = (torch.zeros(B, 1, N, D, device="cuda", dtype=torch.float16) for _ in range(2))
    q[..., 0] = 1.0
    k[:, :, 0, 0] = 18.375
    v[:, :, 1:] = (torch.rand(B, 1, N - 1, D, device="cuda", generator=g) + 1).half()
    pos = torch.arange(N - T, N, device="cuda")
    s = q.double() @ k.double().transpose(-1, -2)
    w = s.masked_fill(torch.arange(N, device="cuda") > pos[:, None], -INF).softmax(-1)
    out = w @ v.double()
    u = 2.0 ** -11
    return q, k, v, out, u * out + 2.0 ** -25 + u * out + 2.0 ** -32 * (pos[:, None] + 1) * 2 + 2.0 ** -20 * out


# sequences that a CTA covers alone, and one that is cut: only the piece with the heavy token has light weights then
@pytest.mark.parametrize("B,D,N", [(300, 64, 2000), (200, 128, 700), (200, 256, 1500), (1, 64, 60000)])
def test_decode_keeps_light_f16_weights(B, D, N):
    q, k, v, out, bound = light_tokens(B, 1, D, N, D)
    got, lse = K().decode_sdpa(q[:, :, 0], k, v, 1.0, return_lse=True)
    K().device_status()
    assert ((got.double() - out[:, :, 0]).abs() <= bound[:, :, 0]).all()
    want = math.log(math.exp(18.375) + N - 1)
    assert ((lse.double() - want).abs() <= 2.0 ** -20 * want).all()


@pytest.mark.parametrize("T,D,N", [(130, 64, 1000), (300, 128, 700), (140, 256, 1500), (2, 128, 1500)])
def test_prompt_keeps_light_f16_weights(T, D, N):
    """As many sequences as there are whole units to show it in."""
    q, k, v, out, bound = light_tokens(40, T, D, N, D)
    got, lse = K().prompt_sdpa(q, k, v, 1.0, return_lse=True)
    K().device_status()
    assert ((got.double() - out).abs() <= bound).all()
    want = torch.log(math.exp(18.375) + torch.arange(N - T, N, device="cuda").double())
    assert ((lse.double() - want).abs() <= 2.0 ** -20 * want).all()


@pytest.mark.parametrize("Hq,Hkv,D,N,page", [(4, 2, 64, 300, 16), (8, 1, 128, 300, 0), (16, 2, 256, 20000, 0)])
def test_output_in_place_of_the_queries(Hq, Hkv, D, N, page):
    from swiftlm_b200 import _lib
    x = Problem(2, Hq, Hkv, 150, D, N, "bf16", page, [N, N - 7], [150, 70], seed=D)
    args = dict(q_len=x.q_len, kv_len=x.kv_len, page_table=x.table)
    want = K().prompt_sdpa(x.q, x.k, x.v, x.scale, out=x.q.clone(), **args)
    q = x.q.clone()
    assert K().prompt_sdpa(q, x.k, x.v, x.scale, out=q, **args) is q and torch.equal(q, want)
    one = x.q[:, :, 0].contiguous()
    args.pop("q_len")
    want = K().decode_sdpa(one, x.k, x.v, x.scale, **args)
    assert K().decode_sdpa(one, x.k, x.v, x.scale, out=one, **args) is one and torch.equal(one, want)
    both = torch.zeros(2 * one.numel(), dtype=x.dt, device="cuda")
    launches = K().launch_count()
    with pytest.raises(_lib.DFlashError):                  # half of it
        K().decode_sdpa(both[:one.numel()].view_as(one), x.k, x.v, x.scale, out=both[D:D + one.numel()].view_as(one), **args)
    assert K().launch_count() == launches
    K().device_status()


def test_evict_between_masses_in_each_others_gaps():
    """mass and mass_out as two columns of one array: rows of 50 every 128, 64 apart."""
    from swiftlm_b200 import _lib
    B, Hkv, D, N, budget = 3, 2, 64, 50, 20
    x = Problem(B, Hkv, Hkv, 1, D, N, "bf16", 0, [50, 31, 7], seed=1, junk=2.0)
    array = torch.rand(B, Hkv, 128, device="cuda")
    before, mass = array.clone(), array[:, :, :N].contiguous()
    k, v, lens = x.k.clone(), x.v.clone(), x.kv_len.clone()
    want = torch.zeros_like(mass)
    K().kv_evict(k, v, mass, lens, budget, 5, 2, mass_out=want)
    out_lens = torch.zeros_like(x.kv_len)
    L = _lib.lib()
    need = L.dflash_kv_evict_workspace_bytes(B, Hkv, N, budget)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    _lib.check(L.dflash_kv_evict(x.k.data_ptr(), x.v.data_ptr(), None, x.kv_len.data_ptr(), array.data_ptr(), out_lens.data_ptr(),
                                 array.data_ptr() + 4 * 64, None, ws.data_ptr(), need, B, Hkv, D, N, 0, 0, 0, 128, budget, 5, 2,
                                 _lib.BF16, torch.cuda.current_stream().cuda_stream))
    K().device_status()
    assert torch.equal(x.k, k) and torch.equal(x.v, v) and torch.equal(out_lens, lens)
    for b, n in enumerate([50, 31, 7]):
        assert torch.equal(array[b, :, 64:64 + n], want[b, :, :n])
        before[b, :, 64:64 + n] = array[b, :, 64:64 + n]
    assert torch.equal(array, before)


@pytest.mark.parametrize("B,Hq,Hkv,D,N,page,window", [
    (32, 16, 2, 64, 6000, 0, 0),          # a block of the joining kernel goes through several runs of 256 keys
    (40, 20, 4, 128, 5000, 16, 3000),
    (33, 40, 2, 64, 3000, 0, 0),          # the same with two groups of heads
])
def test_decode_weights_of_large_batches(B, Hq, Hkv, D, N, page, window):
    lens = [(N * (3 + 5 * b % 17)) // 19 for b in range(B - 2)] + [0, N]
    x = Problem(B, Hq, Hkv, 1, D, N, "bf16", page, lens, seed=B)
    out, lse, mass = x.want(window, 7)
    m = torch.zeros(B, Hkv, N if not page else x.table.shape[1] * page, device="cuda")
    got, z = K().decode_sdpa(x.q[:, :, 0], x.k, x.v, x.scale, kv_len=x.kv_len, page_table=x.table, window=window, sinks=7, mass=m,
                             return_lse=True)
    K().device_status()
    live = x.kv_len > 0
    x.close(got[live], out[live, :, 0])
    x.close_lse(z, lse[:, :, 0])
    x.close_mass(m[:, :, :N], mass)


# (sequence, unit of a row) pairs around 2048, the most whose costs the plan keeps in shared memory
@pytest.mark.parametrize("B,T", [(682, 130), (1024, 70), (683, 130), (2300, 20)])
def test_prompts_around_the_plans_table(B, T):
    g = torch.Generator().manual_seed(B)
    rows = torch.randint(0, T + 1, (B,), generator=g).tolist()
    lens = [r + int(torch.randint(0, 11, (1,), generator=g)) for r in rows]
    rows[-1] = lens[-1] = 0
    x = Problem(B, 4, 1, T, 64, T + 10, "f16", 0, lens, rows, seed=B)  # units of 64 tokens
    x.q[:, :] = x.q[:, :1]                                              # one head four times: a quarter of the oracle's work
    y = Problem(B, 1, 1, T, 64, T + 10, "f16", 0, lens, rows, seed=B)
    y.q, y.kd, y.vd = x.q[:, :1], x.kd, x.vd
    want, want_lse, mass = y.want(17, 3)
    got, z = K().prompt_sdpa(x.q, x.k, x.v, x.scale, q_len=x.q_len, kv_len=x.kv_len, window=17, sinks=3, return_lse=True,
                             out=torch.zeros_like(x.q))
    for h in range(4):
        x.close(got[:, h:h + 1], want)
        x.close_lse(z[:, h:h + 1], want_lse)
    m = torch.zeros(B, 1, T + 10, device="cuda")
    K().attention_mass(x.q, x.k, z, x.scale, m, q_len=x.q_len, kv_len=x.kv_len, window=17, sinks=3)
    K().device_status()
    assert ((m.double() - 4 * mass).abs() <= 4 * (4e-4 * mass + 1e-7) + 4e-4 * 4 * mass).all()      # the lse's error and the scores'


@pytest.mark.parametrize("B,N", [(64, 8190), (70, 8000), (683, 700), (2049, 200)])
def test_weights_around_the_plans_table(B, N):
    g = torch.Generator().manual_seed(N)
    lens = torch.randint(0, N + 1, (B,), generator=g).tolist()
    lens[0], lens[1] = N, 0
    rows = [min(3, n) for n in lens]
    x = Problem(B, 1, 1, 3, 64, N, "bf16", 0, lens, rows, seed=B)
    lse = x.want()[1].float()
    want = x.want(lse_in=lse)[2]
    m = torch.zeros(B, 1, N, device="cuda")
    K().attention_mass(x.q, x.k, lse, x.scale, m, q_len=x.q_len, kv_len=x.kv_len)
    K().device_status()
    x.close_mass(m, want)


@pytest.mark.parametrize("Hq,Hkv,T,D,N,page,window,sinks", [
    (4, 1, 4100, 128, 4100, 0, 0, 0),                      # causal prompts of thousands of tokens
    (4, 2, 4097, 64, 4200, 64, 0, 0),
    (4, 1, 2500, 64, 5001, 0, 700, 64),
    (2, 1, 2049, 256, 4000, 256, 0, 0),
    (8, 2, 40, 128, 30000, 128, 0, 0),                     # a short turn over a long cache
    (8, 2, 33, 256, 20011, 0, 0, 0),
    (16, 2, 65, 64, 30001, 256, 0, 0),
])
def test_long_prompts_and_short_turns(Hq, Hkv, T, D, N, page, window, sinks):
    x = Problem(1, Hq, Hkv, T, D, N, "bf16", page, seed=T + D)
    args = dict(page_table=x.table, window=window, sinks=sinks, n_max=N)
    want, want_lse, _ = x.want(window, sinks)
    got, z = K().prompt_sdpa(x.q, x.k, x.v, x.scale, kv_len=x.kv_len, return_lse=True, **args)
    x.close(got, want)
    x.close_lse(z, want_lse)
    m = torch.zeros(1, Hkv, N, device="cuda")
    K().attention_mass(x.q, x.k, z, x.scale, m, kv_len=x.kv_len, **args)
    K().device_status()
    x.close_mass(m, x.want(window, sinks, lse_in=z)[2])


@pytest.mark.parametrize("B,Hkv,D,N,page,budget", [(6, 2, 64, 9000, 32, 3000), (3, 1, 256, 20000, 0, 17000)])
def test_evict_of_many_fp32_rows(B, Hkv, D, N, page, budget):
    from tests.test_gpu_cache_attention import TYPES, evict_reference
    TYPES.setdefault("f32", torch.float32)
    x = Problem(B, Hkv, Hkv, 1, D, N, "f32", page, [N - 500 * b for b in range(B)], seed=N, junk=2.0)
    mass = torch.randint(0, 200, (B, Hkv, N if not page else x.table.shape[1] * page), device="cuda").float()     # many ties
    places = evict_reference(x, mass.cpu(), budget, 600, 4)
    kept = torch.empty(B, Hkv, budget, dtype=torch.int32, device="cuda")
    K().kv_evict(x.k, x.v, mass, x.kv_len, budget, 600, 4, page_table=x.table, kept=kept)
    K().device_status()
    at = torch.arange(budget, device="cuda")
    for b in range(B):
        for h in range(Hkv):
            p = places[b * Hkv + h]
            assert kept[b, h].tolist() == p
            for pool, dense in ((x.k, x.kd), (x.v, x.vd)):
                rows = pool[b, h, :budget] if not page else pool[x.table[b, at // page].long(), h, at % page]
                assert torch.equal(rows, dense[b, h, p])
