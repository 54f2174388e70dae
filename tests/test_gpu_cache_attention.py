"""The operators on the KV cache outside the verify cycle (one-token attention, prompt attention, accumulated weights,
eviction) against their definitions in 64 bits.

Tolerances, from the arithmetic: the kernels round the weights to the inputs' type before P V (half a step u = eps / 2
each) and the output once more, so |out - want| <= u |want| + u sum_n p_n |v_n| + fp32 slack <= u |want| + u max|v| + slack.
Scores are fp32 sums of D exact products: |ds| <= D * 2^-24 * sum|q k| scale, a relative error of that size in the
weights; the slack SCORE covers it with the sizes used here (|q.k| sums below 400 * scale 1/16, D <= 256: 4e-4).
lse and mass carry the score error only (and 2^-22 of the exponential).  A whole number or a moved byte is exact."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

SCORE = 4e-4
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def K():
    from swiftlm_b200 import kernels
    return kernels


class Problem:
    """Random q, k, v behind a dense cache or a shuffled page pool.  `junk` fills everything behind the lengths and the pages
    that belong to nobody."""

    def __init__(self, B, Hq, Hkv, T, D, N, dtype="bf16", page=0, kv_len=None, q_len=None, seed=0, junk=float("nan"), spread=1.0):
        g = torch.Generator(device="cuda").manual_seed(1000 + seed)
        dt = TYPES[dtype]
        self.B, self.Hq, self.Hkv, self.T, self.D, self.N, self.dt = B, Hq, Hkv, T, D, N, dt
        self.scale = 1.0 / math.sqrt(D)
        rn = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dt)  # noqa: E731
        self.q = rn(B, Hq, T, D) * spread
        self.kd, self.vd = rn(B, Hkv, N, D), rn(B, Hkv, N, D)
        self.kv = [N] * B if kv_len is None else list(kv_len)
        self.ql = [T] * B if q_len is None else list(q_len)
        self.kv_len = torch.tensor(self.kv, dtype=torch.int32, device="cuda")
        self.q_len = torch.tensor(self.ql, dtype=torch.int32, device="cuda")
        kd, vd = self.kd.clone(), self.vd.clone()
        for b in range(B):
            kd[b, :, max(self.kv[b], 0):] = junk
            vd[b, :, max(self.kv[b], 0):] = junk
        self.page = page
        if page:
            pages = -(-N // page)
            perm = torch.randperm(B * pages + 2, generator=g, device="cuda")[:B * pages].view(B, pages)
            self.table = perm.to(torch.int32)
            self.k = torch.full((B * pages + 2, Hkv, page, D), junk, dtype=dt, device="cuda")
            self.v = self.k.clone()
            for b in range(B):
                for i in range(pages):
                    rows = min(page, N - i * page)
                    self.k[perm[b, i], :, :rows] = kd[b, :, i * page:i * page + rows]
                    self.v[perm[b, i], :, :rows] = vd[b, :, i * page:i * page + rows]
        else:
            self.table, self.k, self.v = None, kd, vd

    def seen(self, b, window, sinks):
        n, t = self.kv[b], self.ql[b]
        p = torch.arange(n - t, n, device="cuda")[:, None]
        j = torch.arange(n, device="cuda")[None]
        ok = j <= p
        if window:
            ok &= (j > p - window) | (j < sinks)
        return ok

    def want(self, window=0, sinks=0, scale=None, lse_in=None):
        """(out, lse, mass) in 64 bits; rows not in use: out nan, lse -inf."""
        scale = self.scale if scale is None else scale
        out = torch.full((self.B, self.Hq, self.T, self.D), float("nan"), dtype=torch.float64, device="cuda")
        lse = torch.full((self.B, self.Hq, self.T), -math.inf, dtype=torch.float64, device="cuda")
        mass = torch.zeros(self.B, self.Hkv, self.N, dtype=torch.float64, device="cuda")
        G = self.Hq // self.Hkv
        for b in range(self.B):
            n, t = self.kv[b], self.ql[b]
            ok = self.seen(b, window, sinks)
            for h in range(self.Hq):
                s = self.q[b, h, :t].double() @ self.kd[b, h // G, :n].double().T * scale
                s = s.masked_fill(~ok, -math.inf)
                z = torch.logsumexp(s, -1) if n else torch.full((t,), -math.inf, dtype=torch.float64, device="cuda")
                used = z if lse_in is None else lse_in[b, h, :t].double()
                w = torch.where(ok & (used > -math.inf)[:, None], torch.exp(s - used[:, None]), torch.zeros_like(s))
                lse[b, h, :t] = z
                out[b, h, :t] = w @ self.vd[b, h // G, :n].double()
                mass[b, h // G, :n] += w.sum(0)
        return out, lse, mass

    def close(self, got, want):
        u = torch.finfo(self.dt).eps / 2
        bound = u * want.abs() + u * self.vd.double().abs().max() + SCORE
        live = ~torch.isnan(want)
        d = (got.double() - want)[live].abs()
        assert torch.isfinite(got[live]).all()
        assert (d <= bound[live]).all(), float((d / bound[live]).max())

    def close_lse(self, got, want):
        assert torch.equal(got == -math.inf, want == -math.inf)
        live = want > -math.inf
        assert ((got.double() - want)[live].abs() <= SCORE + 2.0 ** -22 * want[live].abs()).all()

    def close_mass(self, got, want):
        d = (got.double() - want).abs()
        assert (d <= SCORE * want + 1e-7).all(), float((d / (SCORE * want + 1e-7)).max())


DECODE = [
    # B, Hq, Hkv, D, N, dtype, page, lengths, window, sinks
    (1, 1, 1, 64, 1, "bf16", 0, None, 0, 0),
    (1, 16, 2, 256, 517, "bf16", 0, None, 0, 0),
    (2, 16, 2, 256, 129, "f16", 0, [1, 129], 0, 0),
    (5, 12, 4, 64, 331, "f16", 16, [331, 0, 17, 64, 1], 0, 0),
    (3, 10, 2, 128, 1000, "bf16", 48, [1000, 47, 49], 0, 0),
    (4, 32, 8, 128, 2500, "f16", 64, [2500, 64, 1088, 1089], 1024, 64),
    (3, 24, 2, 256, 700, "bf16", 128, [700, 300, 5], 100, 7),
    (2, 32, 2, 128, 600, "bf16", 256, [600, 599], 1, 0),
    (2, 40, 1, 64, 300, "bf16", 0, [300, 33], 33, 1),
    (1, 48, 2, 256, 4099, "bf16", 256, None, 0, 0),
    (1, 8, 8, 128, 20000, "f16", 0, None, 0, 0),
    (70, 4, 2, 64, 80, "bf16", 16, [(7 * i) % 81 for i in range(70)], 0, 0),
    (2, 3, 3, 256, 513, "bf16", 0, [513, 512], 64, 512),
]


@pytest.mark.parametrize("B,Hq,Hkv,D,N,dtype,page,lens,window,sinks", DECODE)
@pytest.mark.parametrize("with_mass", [False, True])
def test_decode_matches_the_definition(B, Hq, Hkv, D, N, dtype, page, lens, window, sinks, with_mass):
    x = Problem(B, Hq, Hkv, 1, D, N, dtype, page, lens, seed=B * N + D)
    out, lse, mass = x.want(window, sinks)
    cap = x.N if not page else x.table.shape[1] * page
    m = torch.full((B, Hkv, cap + 3), 0.25, device="cuda") if with_mass else None
    got, z = K().decode_sdpa(x.q[:, :, 0], x.k, x.v, x.scale, kv_len=x.kv_len, page_table=x.table, window=window, sinks=sinks,
                             mass=m, return_lse=True)
    K().device_status()
    empty = x.kv_len == 0
    assert (got[empty] == 0).all() and (z[empty] == -math.inf).all()
    x.close(got[~empty], out[~empty, :, 0])
    x.close_lse(z, lse[:, :, 0])
    if with_mass:
        x.close_mass(m[:, :, :N] - 0.25, mass)
        assert (m[:, :, N:] == 0.25).all()
        for b in range(B):
            assert (m[b, :, x.kv[b]:] == 0.25).all()
    again = K().decode_sdpa(x.q[:, :, 0], x.k, x.v, x.scale, kv_len=x.kv_len, page_table=x.table, window=window, sinks=sinks)
    assert torch.equal(again, got)                    # the same bits, with and without the other outputs


PROMPT = [
    # B, Hq, Hkv, T, D, N, dtype, page, kv_len, q_len, window, sinks
    (1, 1, 1, 1, 64, 1, "bf16", 0, None, None, 0, 0),
    (1, 4, 2, 17, 128, 17, "f16", 0, None, None, 0, 0),
    (2, 16, 2, 128, 256, 128, "bf16", 0, None, None, 0, 0),
    (2, 16, 2, 129, 256, 400, "bf16", 128, [400, 129], None, 0, 0),
    (3, 12, 4, 193, 64, 331, "f16", 16, [331, 193, 200], [193, 1, 65], 0, 0),
    (2, 8, 8, 300, 128, 700, "bf16", 48, [700, 300], [300, 299], 100, 7),
    (1, 8, 2, 1000, 128, 1000, "f16", 0, None, None, 256, 64),
    (2, 10, 2, 333, 256, 1500, "bf16", 256, [1500, 333], None, 200, 5),
    (1, 16, 2, 9, 256, 5000, "bf16", 256, None, None, 0, 0),
    (4, 3, 1, 40, 64, 90, "bf16", 16, [90, 10, 0, 40], [40, 40, 40, 0], 0, 0),   # rows in front of the first token, no rows
    (1, 2, 1, 513, 128, 513, "bf16", 0, None, None, 1, 0),
    (1, 2, 1, 257, 64, 2000, "bf16", 64, None, None, 64, 300),
    (1, 4, 4, 640, 64, 640, "f16", 0, None, None, 0, 0),
    (3, 16, 2, 300, 256, 300, "bf16", 256, [300, 100, 257], [300, 100, 257], 0, 0),      # several query tiles, one key tile of two
    (2, 48, 1, 50, 128, 120, "bf16", 0, [120, 60], [50, 50], 0, 0),                      # 2 tokens a query tile
    (1, 260, 2, 6, 64, 70, "f16", 0, None, None, 0, 0),                                  # more heads in a group than rows in a tile
    (9, 6, 2, 5, 128, 50, "f16", 0, [50, 5, 7, 49, 33, 16, 17, 5, 5], None, 3, 2),
]


@pytest.mark.parametrize("B,Hq,Hkv,T,D,N,dtype,page,lens,rows,window,sinks", PROMPT)
def test_prompt_matches_the_definition(B, Hq, Hkv, T, D, N, dtype, page, lens, rows, window, sinks):
    x = Problem(B, Hq, Hkv, T, D, N, dtype, page, lens, rows, seed=B * N + D + T)
    want, want_lse, _ = x.want(window, sinks)
    out = torch.full_like(x.q, 3.0)
    got, z = K().prompt_sdpa(x.q, x.k, x.v, x.scale, q_len=x.q_len, kv_len=x.kv_len, page_table=x.table, window=window,
                             sinks=sinks, return_lse=True, out=out)
    K().device_status()
    assert got is out
    x.close(got, want)
    x.close_lse(z, want_lse)
    for b in range(B):
        assert (got[b, :, x.ql[b]:] == 3.0).all()                          # rows behind the last query
        assert (got[b, :, :max(0, x.ql[b] - x.kv[b])] == 0).all()          # rows in front of the first token
    again = K().prompt_sdpa(x.q, x.k, x.v, x.scale, q_len=x.q_len, kv_len=x.kv_len, page_table=x.table, window=window, sinks=sinks,
                            out=torch.full_like(x.q, 3.0))
    assert torch.equal(again, got)


@pytest.mark.parametrize("B,Hq,Hkv,T,D,N,dtype,page,lens,rows,window,sinks", PROMPT)
def test_mass_matches_the_definition(B, Hq, Hkv, T, D, N, dtype, page, lens, rows, window, sinks):
    x = Problem(B, Hq, Hkv, T, D, N, dtype, page, lens, rows, seed=B * N + D + T)
    lse = x.want(window, sinks)[1].float()
    want = x.want(window, sinks, lse_in=lse)[2]
    cap = N if not page else x.table.shape[1] * page
    m = torch.full((B, Hkv, cap + 1), 0.5, device="cuda")
    junk = lse.clone()
    for b in range(B):
        junk[b, :, x.ql[b]:] = float("nan")                                 # not read
    for k in range(2):
        K().attention_mass(x.q, x.k, junk, x.scale, m, q_len=x.q_len, kv_len=x.kv_len, page_table=x.table, window=window, sinks=sinks)
        K().device_status()
        for b in range(B):
            assert (m[b, :, x.kv[b]:] == 0.5).all()
        x.close_mass((m[:, :, :N] - 0.5) / (k + 1), want)


def test_small_and_large_scales():
    x = Problem(2, 8, 2, 40, 128, 300, "bf16", 64, [300, 100], seed=5, spread=8.0)
    for scale in (1e-12, 0.02, 0.25):
        want, want_lse, _ = x.want(scale=scale)
        got, z = K().prompt_sdpa(x.q, x.k, x.v, scale, q_len=x.q_len, kv_len=x.kv_len, page_table=x.table, return_lse=True)
        # products up to 8 * 128 * 4 * 4 in size: fp32 sums of 128 terms are off by 2^-24 * 128 * 8 * 128 * scale
        slack = 2.0 ** -24 * 128 * 8 * 128 * abs(scale)
        u = torch.finfo(x.dt).eps / 2
        assert ((z.double() - want_lse).abs() <= slack + 2.0 ** -21 * want_lse.abs() + 1e-6).all()
        assert ((got.double() - want).abs() <= u * want.abs() + (u + 2 * slack) * x.vd.double().abs().max() + SCORE).all()
        d = K().decode_sdpa(x.q[:, :, -1].contiguous(), x.k, x.v, scale, kv_len=x.kv_len, page_table=x.table)
        assert ((d.double() - want[:, :, -1]).abs() <= u * want[:, :, -1].abs() + (u + 2 * slack) * x.vd.double().abs().max() + SCORE).all()


def evict_reference(x, mass, budget, recent, sinks):
    """Per head, by sorting: lists of the places that stay."""
    places = []
    for b, n in enumerate(x.kv):
        for h in range(x.Hkv):
            if n <= budget:
                places.append(list(range(n)))
                continue
            w = mass[b, h, :n].tolist()
            key = [math.inf if math.isnan(v) else v for v in w]
            nan = [math.isnan(v) for v in w]
            middle = sorted(range(sinks, n - recent), key=lambda i: (not nan[i], -key[i], i))
            places.append(sorted(list(range(sinks)) + list(range(n - recent, n)) + middle[:budget - sinks - recent]))
    return places


EVICT = [
    # B, Hkv, D, N, dtype, page, lengths, budget, recent, sinks
    (1, 1, 64, 2, "bf16", 0, None, 1, 0, 0),
    (2, 2, 256, 1104, "bf16", 128, None, 1088, 512, 64),
    (4, 3, 64, 700, "f16", 16, [700, 65, 64, 0], 64, 20, 5),
    (3, 1, 128, 5000, "bf16", 48, [5000, 4999, 100], 2000, 0, 0),
    (2, 2, 128, 3000, "f32", 0, [3000, 1500], 1024, 1000, 24),        # nothing but sinks and recent tokens stays
    (1, 2, 256, 4097, "bf16", 7, None, 4096, 1, 1),
    (2, 8, 8, 300, "f16", 0, [300, 299], 17, 3, 2),
    (1, 1, 128, 40000, "bf16", 256, None, 4096, 1024, 64),
]


@pytest.mark.parametrize("B,Hkv,D,N,dtype,page,lens,budget,recent,sinks", EVICT)
@pytest.mark.parametrize("weights", ["skewed", "ties", "odd"])
@pytest.mark.parametrize("in_place", [False, True])
def test_evict_matches_sorting(B, Hkv, D, N, dtype, page, lens, budget, recent, sinks, weights, in_place):
    TYPES.setdefault("f32", torch.float32)
    x = Problem(B, Hkv, Hkv, 1, D, N, dtype, page, lens, seed=N + budget, junk=2.0)
    g = torch.Generator(device="cuda").manual_seed(9)
    cap = N if not page else x.table.shape[1] * page
    mass = torch.empty(B, Hkv, cap, device="cuda").exponential_(generator=g) ** 3
    if weights == "ties":
        mass = torch.randint(0, 4, mass.shape, device="cuda", generator=g).float()
    if weights == "odd":                               # signs, zeros of both signs, infinities and NaN
        pick = torch.randint(0, 7, mass.shape, device="cuda", generator=g)
        for i, v in enumerate((0.0, -0.0, -1.5, math.inf, -math.inf, math.nan)):
            mass[pick == i] = v
    before = mass.clone()
    places = evict_reference(x, mass.cpu(), budget, recent, sinks)
    k0, v0 = x.k.clone(), x.v.clone()
    kept = torch.full((B, Hkv, budget), 77, dtype=torch.int32, device="cuda")
    out_mass = mass if in_place else torch.full_like(mass, 9.0)
    lens_out = x.kv_len if in_place else torch.zeros_like(x.kv_len)
    got = K().kv_evict(x.k, x.v, mass, x.kv_len, budget, recent, sinks, page_table=x.table, kv_len_out=lens_out, mass_out=out_mass,
                       kept=None if in_place else kept)
    K().device_status()
    assert got is lens_out and got.tolist() == [min(n, budget) for n in x.kv]
    if not in_place:
        assert torch.equal(torch.nan_to_num(mass), torch.nan_to_num(before))

    def rows(pool, b, h, idx):
        idx = torch.tensor(idx, dtype=torch.long, device="cuda")
        return pool[b, h, idx] if not page else pool[x.table[b, idx // page].long(), h, idx % page]

    expect_k, expect_v = k0.clone(), v0.clone()
    for b in range(B):
        for h in range(Hkv):
            p, n = places[b * Hkv + h], x.kv[b]
            left = len(p)
            to = torch.arange(left, device="cuda")
            for e, src in ((expect_k, k0), (expect_v, v0)):
                if page:
                    e[x.table[b, to // page].long(), h, to % page] = rows(src, b, h, p)
                else:
                    e[b, h, :left] = rows(src, b, h, p)
            m = out_mass[b, h]
            torch.testing.assert_close(m[:left], before[b, h, torch.tensor(p, dtype=torch.long, device="cuda")], rtol=0, atol=0, equal_nan=True)
            assert (m[left:n] == 0).all()
            tail = before[b, h, n:] if in_place else torch.full_like(m[n:], 9.0)
            torch.testing.assert_close(m[n:], tail, rtol=0, atol=0, equal_nan=True)
            if not in_place:
                assert kept[b, h, :left].tolist() == p and (kept[b, h, left:] == -1).all()
    assert torch.equal(x.k, expect_k) and torch.equal(x.v, expect_v)        # byte movement; everything else as it was


def test_lengths_out_of_range_are_clamped_and_reported():
    from swiftlm_b200 import _lib
    x = Problem(3, 8, 2, 20, 128, 200, "bf16", 64, [200, 120, 0], [20, 20, 0], seed=3, junk=1.0)
    want = K().prompt_sdpa(x.q, x.k, x.v, x.scale, q_len=x.q_len, kv_len=x.kv_len, page_table=x.table, n_max=200, out=torch.zeros_like(x.q))
    K().device_status()
    bad_kv = torch.tensor([2 ** 30, 120, -5], dtype=torch.int32, device="cuda")
    bad_q = torch.tensor([21, 20, -1], dtype=torch.int32, device="cuda")
    got = K().prompt_sdpa(x.q, x.k, x.v, x.scale, q_len=bad_q, kv_len=bad_kv, page_table=x.table, n_max=200, out=torch.zeros_like(x.q))
    with pytest.raises(_lib.DFlashError) as e:
        K().device_status()
    assert e.value.status == _lib.ERR_DEVICE_DATA and torch.equal(got, want)
    one = K().decode_sdpa(x.q[:, :, 0], x.k, x.v, x.scale, kv_len=x.kv_len, page_table=x.table, n_max=200)
    K().device_status()
    two = K().decode_sdpa(x.q[:, :, 0], x.k, x.v, x.scale, kv_len=bad_kv, page_table=x.table, n_max=200)
    with pytest.raises(_lib.DFlashError):
        K().device_status()
    assert torch.equal(one, two)
    m = torch.rand(3, 2, 256, device="cuda")
    lens = bad_kv.clone()
    K().kv_evict(x.k, x.v, m, lens, 64, 8, 4, page_table=x.table, n_max=200)
    with pytest.raises(_lib.DFlashError):
        K().device_status()
    assert lens.tolist() == [64, 64, 0]


def test_page_ids_outside_the_pool_read_as_zeros_and_are_reported():
    from swiftlm_b200 import _lib
    x = Problem(2, 8, 2, 24, 128, 320, "bf16", 64, None, None, seed=4, junk=1.0)
    lse = x.want()[1].float()
    for bad_id in (-1, x.k.shape[0], 2 ** 30):
        table = x.table.clone()
        table[1, 2] = bad_id
        y = Problem(2, 8, 2, 24, 128, 320, "bf16", 64, None, None, seed=4, junk=1.0)
        y.kd[1, :, 128:192] = 0
        y.vd[1, :, 128:192] = 0
        want, want_lse, _ = y.want()
        got, z = K().prompt_sdpa(x.q, x.k, x.v, x.scale, page_table=table, n_max=320, return_lse=True)
        with pytest.raises(_lib.DFlashError) as e:
            K().device_status()
        assert e.value.status == _lib.ERR_DEVICE_DATA
        y.close(got, want)
        y.close_lse(z, want_lse)
        d = K().decode_sdpa(x.q[:, :, -1].contiguous(), x.k, x.v, x.scale, page_table=table, n_max=320)
        with pytest.raises(_lib.DFlashError):
            K().device_status()
        y.close(d, want[:, :, -1])
        m = torch.zeros(2, 2, 320, device="cuda")
        K().attention_mass(x.q, x.k, lse, x.scale, m, page_table=table, n_max=320)
        with pytest.raises(_lib.DFlashError):
            K().device_status()
        y.close_mass(m, y.want(lse_in=lse)[2])
