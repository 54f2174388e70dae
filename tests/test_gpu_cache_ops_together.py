"""The cache operators as they are used together: prompts, their weights, eviction and plain decoding over one paged cache,
against growing arrays in 64 bits; captured and replayed graphs, side streams, calls back to back, large offsets.
Tolerances as in test_gpu_cache_attention.py: u per rounding of a weight (times the largest value) and of the output."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
U = torch.finfo(BF).eps / 2


def K():
    from swiftlm_b200 import kernels
    return kernels


def attend64(q, k, v, scale, window=0, sinks=0):
    """q [Hq,T,D] are the last T of the n tokens k, v [Hkv,n,D]; (out, weights) in 64 bits."""
    Hq, T, D = q.shape
    Hkv, n, _ = k.shape
    kk, vv = k.double().repeat_interleave(Hq // Hkv, 0), v.double().repeat_interleave(Hq // Hkv, 0)
    s = q.double() @ kk.transpose(-1, -2) * scale
    p, j = torch.arange(n - T, n, device=q.device)[:, None], torch.arange(n, device=q.device)[None]
    ok = j <= p
    if window:
        ok &= (j > p - window) | (j < sinks)
    w = s.masked_fill(~ok, -math.inf).softmax(-1)
    return w @ vv, w


def close_mass(got, want):
    d = (got.double() - want).abs() - 4e-4 * want - 1e-6
    assert float(d.max()) <= 0, float(d.max())


def close(got, want, vmax=6.0):
    d = (got.double() - want).abs()
    assert torch.isfinite(got).all() and (d <= U * want.abs() + U * vmax + 4e-4).all(), float(d.max())


@pytest.mark.parametrize("page,D,Hq,Hkv", [(16, 64, 6, 2), (64, 128, 8, 2), (256, 256, 16, 2)])
def test_prompt_weights_eviction_and_decoding_over_one_cache(page, D, Hq, Hkv):
    from swiftlm_b200.kv_cache import PagedKVCache
    B, P, budget, recent, sinks = 3, 300, 128, 32, 4
    g = torch.Generator(device="cuda").manual_seed(D)
    rn = lambda *s: torch.randn(*s, device="cuda", generator=g).to(BF)  # noqa: E731
    pages = -(-(P + 64) // page)
    cache = PagedKVCache(B, Hkv, D, page, num_pages=B * pages + 1, max_pages=pages, track_mass=True)
    cache.k_pool.fill_(float("nan"))                       # nothing but appended rows may count
    cache.v_pool.fill_(float("nan"))
    scale, lens = D ** -0.5, [300, 100, 257]
    k, v, q = rn(B, Hkv, P, D), rn(B, Hkv, P, D), rn(B, Hq, P, D)
    cache.extend(k, v, lens)
    ql = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out, lse = cache.attend_prompt(q, scale, q_len=ql, return_lse=True)
    cache.add_mass(q, lse, scale, q_len=ql)
    keys = [k[b, :, :lens[b]] for b in range(B)]
    vals = [v[b, :, :lens[b]] for b in range(B)]
    mass = []
    for b in range(B):
        want, w = attend64(q[b, :, :lens[b]], keys[b], vals[b], scale)
        close(out[b, :, :lens[b]], want)
        mass.append(w.view(Hkv, -1, lens[b], lens[b]).sum((1, 2)))
        close_mass(cache.mass[b, :, :lens[b]], mass[b])
        mass[b] = cache.mass[b, :, :lens[b]].clone()        # the choice below goes by the values that the cache has
    before = cache.free_pages
    for step in range(6):
        if step in (0, 4):
            cache.evict(budget, recent, sinks)
            for b in range(B):
                n = keys[b].shape[1]
                if n <= budget:
                    continue
                kb, vb, mb = [], [], []
                for h in range(Hkv):
                    order = torch.sort(mass[b][h, sinks:n - recent], descending=True, stable=True).indices[:budget - recent - sinks] + sinks
                    idx = torch.cat([torch.arange(sinks, device="cuda"), order.sort().values, torch.arange(n - recent, n, device="cuda")])
                    kb.append(keys[b][h, idx]); vb.append(vals[b][h, idx]); mb.append(mass[b][h, idx])
                keys[b], vals[b], mass[b] = torch.stack(kb), torch.stack(vb), torch.stack(mb)
            assert cache.free_pages >= before
        k1, v1, q1 = rn(B, Hkv, 1, D), rn(B, Hkv, 1, D), rn(B, Hq, D)
        window, s0 = (0, 0) if step < 3 else (50, 4)
        cache.append_block(k1, v1)
        one, z = cache.attend_one(q1, scale, window=window, sinks=s0, return_lse=True)
        cache.commit(torch.ones(B, dtype=torch.int32, device="cuda"))
        for b in range(B):
            keys[b], vals[b] = torch.cat([keys[b], k1[b]], 1), torch.cat([vals[b], v1[b]], 1)
            want, w = attend64(q1[b][:, None], keys[b], vals[b], scale, window, s0)
            close(one[b], want[:, 0])
            n = keys[b].shape[1]
            mass[b] = torch.cat([mass[b], torch.zeros(Hkv, 1, device="cuda")], 1).double() + w.view(Hkv, -1, n).sum(1)
            got = cache.mass[b, :, :n]
            close_mass(got, mass[b])
            mass[b] = got.clone()
    lengths = cache.sync().tolist()
    assert lengths == [x.shape[1] for x in keys]
    for b in range(B):
        gk, gv = cache.gather(b)
        assert torch.equal(gk, keys[b]) and torch.equal(gv, vals[b])
    K().device_status()
    # a verify block still works on what is left, and the weights of the rows it keeps can be added
    if page % 128 == 0:
        kn, vn, qn = rn(B, Hkv, 16, D), rn(B, Hkv, 16, D), rn(B, Hq, 16, D)
        cache.append_block(kn, vn)
        block = cache.attend(qn, scale)
        keep = torch.tensor([16, 3, 1], dtype=torch.int32, device="cuda")
        cache.commit(keep)
        again, lse = cache.attend_prompt(qn, scale, q_len=keep, return_lse=True)
        cache.add_mass(qn, lse, scale, q_len=keep)
        for b, n in enumerate(keep.tolist()):
            want, w = attend64(qn[b, :, :n], torch.cat([keys[b], kn[b, :, :n]], 1), torch.cat([vals[b], vn[b, :, :n]], 1), scale)
            close(block[b, :, :n], want)
            close(again[b, :, :n], want)
            total = lengths[b] + n
            m = torch.cat([mass[b], torch.zeros(Hkv, n, device="cuda")], 1).double() + w.view(Hkv, -1, n, total).sum((1, 2))
            close_mass(cache.mass[b, :, :total], m)
        K().device_status()


def make(seed, B=3, Hq=8, Hkv=2, D=128, N=700, T=40, page=64):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(*s, device="cuda", generator=g).to(BF)  # noqa: E731
    pages = -(-N // page)
    return dict(k=rn(B * pages, Hkv, page, D), v=rn(B * pages, Hkv, page, D), q=rn(B, Hq, T, D), q1=rn(B, Hq, D),
                table=torch.randperm(B * pages, device="cuda", generator=g).view(B, pages).to(torch.int32),
                kv_len=torch.tensor([N, N // 2, 77], dtype=torch.int32, device="cuda"), mass=torch.zeros(B, Hkv, pages * page, device="cuda"),
                scale=D ** -0.5, out=torch.zeros(B, Hq, T, D, dtype=BF, device="cuda"))


def cycle(x):
    """A run of all four on one problem; every result is left in x or returned."""
    one, z = K().decode_sdpa(x["q1"], x["k"], x["v"], x["scale"], kv_len=x["kv_len"], page_table=x["table"], mass=x["mass"], window=300,
                             sinks=5, return_lse=True)
    out, lse = K().prompt_sdpa(x["q"], x["k"], x["v"], x["scale"], kv_len=x["kv_len"], page_table=x["table"], return_lse=True, out=x["out"])
    K().attention_mass(x["q"], x["k"], lse, x["scale"], x["mass"], kv_len=x["kv_len"], page_table=x["table"])
    K().kv_evict(x["k"], x["v"], x["mass"], x["kv_len"], 256, 64, sinks=4, page_table=x["table"])
    return one, z, out, lse


def snapshot(x, results):
    return [t.clone() for t in results] + [x[n].clone() for n in ("k", "v", "mass", "kv_len")]


def test_back_to_back_on_several_streams_gives_the_bits_of_one_at_a_time():
    want = []
    for seed in range(6):
        x = make(seed)
        want.append(snapshot(x, cycle(x)))
        torch.cuda.synchronize()
    xs = [make(seed) for seed in range(6)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for i, x in enumerate(xs):
        with torch.cuda.stream(streams[i % 3]):
            got.append(snapshot(x, cycle(x)))
    torch.cuda.synchronize()
    K().device_status()
    for a, b in zip(got, want):
        for s, t in zip(a, b):
            assert torch.equal(s, t)


def test_two_captured_graphs_replayed_at_once_over_changing_inputs():
    xs = [make(10), make(11)]
    for x in xs:
        cycle(x)                                           # function attributes are set on first use
    torch.cuda.synchronize()
    graphs, results = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            results.append(cycle(x))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in xs]
    for round_ in range(3):
        fresh = [make(20 + 2 * round_ + i) for i in range(2)]
        want = [snapshot(f, cycle(f)) for f in [make(20 + 2 * round_ + i) for i in range(2)]]
        for x, f in zip(xs, fresh):
            for n in ("k", "v", "q", "q1", "table", "kv_len", "mass", "out"):
                x[n].copy_(f[n])
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for x, r, w in zip(xs, results, want):
            for s, t in zip(snapshot(x, r), w):
                assert torch.equal(s, t)
    K().device_status()


def test_more_sequences_than_one_launch_takes():
    B, Hq, Hkv, D, N = 1300, 4, 2, 64, 40
    g = torch.Generator(device="cuda").manual_seed(1)
    rn = lambda *s: torch.randn(*s, device="cuda", generator=g).to(BF)  # noqa: E731
    k, v, q = rn(B, Hkv, N, D), rn(B, Hkv, N, D), rn(B, Hq, D)
    lens = torch.randint(0, N + 1, (B,), device="cuda", generator=g, dtype=torch.int32)
    mass = torch.zeros(B, Hkv, N, device="cuda")
    out = K().decode_sdpa(q, k, v, 0.125, kv_len=lens, mass=mass)
    s = (q.double().view(B, Hkv, 2, 1, D) @ k.double()[:, :, None].transpose(-1, -2) * 0.125)
    s = s.masked_fill(torch.arange(N, device="cuda") >= lens.view(B, 1, 1, 1, 1), -math.inf)
    w = torch.nan_to_num(s.softmax(-1))
    close(out, (w @ v.double()[:, :, None]).view(B, Hq, D))
    close_mass(mass, w.sum((2, 3)))
    p = K().prompt_sdpa(q[:, :, None].contiguous(), k, v, 0.125, kv_len=lens)
    close(p[:, :, 0], (w @ v.double()[:, :, None]).view(B, Hq, D))
    K().device_status()


def test_offsets_past_32_bits():
    """A pool of more than 2^31 elements, read and moved at its far end."""
    Hkv, page, D, pages = 2, 256, 256, 17000
    k, v = (torch.empty(pages, Hkv, page, D, dtype=BF, device="cuda") for _ in range(2))
    g = torch.Generator(device="cuda").manual_seed(2)
    ids = [pages - 1, 3, pages - 2]
    for t in (k, v):
        for i in ids:
            t[i] = torch.randn(Hkv, page, D, device="cuda", generator=g).to(BF)
    q = torch.randn(1, 16, 20, D, device="cuda", generator=g).to(BF)
    table = torch.tensor([ids], dtype=torch.int32, device="cuda")
    n = 700
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    dk, dv = (torch.cat([t[i] for i in ids], 1)[:, :n].clone() for t in (k, v))
    want, w = attend64(q[0], dk, dv, 1 / 16)
    out, lse = K().prompt_sdpa(q, k, v, 1 / 16, kv_len=lens, page_table=table, return_lse=True)
    close(out[0], want)
    one = K().decode_sdpa(q[:, :, -1].contiguous(), k, v, 1 / 16, kv_len=lens, page_table=table)
    close(one[0], want[:, -1])
    mass = torch.zeros(1, Hkv, 3 * page, device="cuda")
    K().attention_mass(q, k, lse, 1 / 16, mass, kv_len=lens, page_table=table)
    m = w.view(Hkv, 8, 20, n).sum((1, 2))
    close_mass(mass[0, :, :n], m)
    kept = torch.empty(1, Hkv, 600, dtype=torch.int32, device="cuda")
    K().kv_evict(k, v, mass, lens, 600, 100, page_table=table, kept=kept)
    for h in range(Hkv):
        idx = kept[0, h].long()
        assert torch.equal(torch.cat([k[i, h] for i in ids])[:600], dk[h, idx])
        assert torch.equal(torch.cat([v[i, h] for i in ids])[:600], dv[h, idx])
    assert lens.item() == 600
    K().device_status()


def test_views_are_taken_and_wrong_tensors_refused():
    from swiftlm_b200 import _lib
    x = make(3)
    base = K().decode_sdpa(x["q1"], x["k"], x["v"], x["scale"], kv_len=x["kv_len"], page_table=x["table"])
    wide = torch.empty(3, 8, 256, dtype=BF, device="cuda")
    wide[..., ::2] = x["q1"]
    assert torch.equal(K().decode_sdpa(wide[..., ::2], x["k"], x["v"], x["scale"], kv_len=x["kv_len"].tolist(), page_table=x["table"].long()), base)
    shifted = torch.empty(3 * 8 * 40 * 128 + 8, dtype=BF, device="cuda")[8:].view(3, 8, 40, 128)      # 16-byte aligned, not 32
    a = K().prompt_sdpa(x["q"], x["k"], x["v"], x["scale"], kv_len=x["kv_len"], page_table=x["table"], out=shifted)
    assert torch.equal(a, K().prompt_sdpa(x["q"], x["k"], x["v"], x["scale"], kv_len=x["kv_len"], page_table=x["table"]))
    bad = [lambda: K().decode_sdpa(x["q"], x["k"], x["v"], x["scale"]),
           lambda: K().decode_sdpa(x["q1"].half(), x["k"], x["v"], x["scale"], page_table=x["table"]),
           lambda: K().decode_sdpa(x["q1"].float(), x["k"].float(), x["v"].float(), x["scale"], page_table=x["table"]),
           lambda: K().decode_sdpa(x["q1"], x["k"], x["v"][:-1], x["scale"], page_table=x["table"]),
           lambda: K().decode_sdpa(x["q1"], x["k"], x["v"], x["scale"], page_table=x["table"][:2]),
           lambda: K().decode_sdpa(x["q1"], x["k"], x["v"], x["scale"], page_table=x["table"], kv_len=x["kv_len"][:2]),
           lambda: K().decode_sdpa(x["q1"], x["k"], x["v"], x["scale"], page_table=x["table"], mass=x["mass"].half()),
           lambda: K().decode_sdpa(x["q1"], x["k"], x["v"], x["scale"], page_table=x["table"], mass=x["mass"][:, :, :500]),
           lambda: K().decode_sdpa(x["q1"], x["k"], x["v"], x["scale"], page_table=x["table"], out=torch.empty_like(x["q"])),
           lambda: K().decode_sdpa(x["q1"], x["k"], x["v"], -1.0, page_table=x["table"]),
           lambda: K().prompt_sdpa(x["q"], x["k"], x["v"], x["scale"], page_table=x["table"], window=-1),
           lambda: K().prompt_sdpa(x["q"][:2], x["k"], x["v"], x["scale"], page_table=x["table"]),
           lambda: K().attention_mass(x["q"], x["k"], torch.zeros(3, 8, 39, device="cuda"), x["scale"], x["mass"], page_table=x["table"]),
           lambda: K().attention_mass(x["q"], x["k"], torch.zeros(3, 8, 40, device="cpu"), x["scale"], x["mass"], page_table=x["table"]),
           lambda: K().kv_evict(x["k"], x["v"], x["mass"], x["kv_len"], 10, 9, sinks=2, page_table=x["table"]),
           lambda: K().kv_evict(x["k"].transpose(1, 2), x["v"].transpose(1, 2), x["mass"], x["kv_len"], 10, 1, page_table=x["table"]),
           lambda: K().kv_evict(x["k"], x["v"], x["mass"], x["kv_len"].long(), 10, 1, page_table=x["table"]),
           lambda: K().kv_evict(x["k"], x["v"], x["mass"], x["kv_len"], 10, 1, page_table=x["table"],
                                kept=torch.empty(3, 2, 9, dtype=torch.int32, device="cuda"))]
    launches = K().launch_count()
    for i, f in enumerate(bad):
        with pytest.raises(_lib.DFlashError):
            f()
            pytest.fail(f"call {i} was taken")
    assert K().launch_count() == launches
    from swiftlm_b200.kv_cache import PagedKVCache
    cache = PagedKVCache(1, 2, 64, 16, num_pages=4, max_pages=4)
    with pytest.raises(RuntimeError):
        cache.evict(8, 2)
    with pytest.raises(RuntimeError):
        cache.attend_one(torch.zeros(1, 2, 64, dtype=BF, device="cuda"), 1.0)


@pytest.mark.gpu
def test_named_arguments_and_scalars_of_other_types():
    import numpy as np
    from swiftlm_b200 import kernels
    torch.manual_seed(5)
    q = torch.randn(2, 4, 3, 64, device="cuda", dtype=torch.bfloat16)
    k, v = (torch.randn(2, 2, 40, 64, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    one = q[:, :, -1].contiguous()
    a = kernels.decode_sdpa(one, k, v, 0.125, window=16, sinks=2)
    b = kernels.decode_sdpa(queries=one, keys=k, values=v, scale=np.float32(0.125), window=np.int64(16), sinks=np.int32(2))
    assert torch.equal(a, b)
    a, lse = kernels.prompt_sdpa(q, k, v, 0.125, window=16, sinks=2, return_lse=True)
    b = kernels.prompt_sdpa(queries=q, keys=k, values=v, scale=torch.tensor(0.125), window=torch.tensor(16), sinks=np.int32(2))
    assert torch.equal(a, b)
    m1, m2 = (torch.zeros(2, 2, 40, device="cuda") for _ in range(2))
    kernels.attention_mass(q, k, lse, 0.125, m1, window=16, sinks=2)
    kernels.attention_mass(queries=q, keys=k, lse=lse, scale=np.float64(0.125), mass=m2, window=np.int64(16), sinks=np.int64(2))
    assert torch.equal(m1, m2)
    n1, n2 = (torch.full((2,), 40, dtype=torch.int32, device="cuda") for _ in range(2))
    k1, v1, k2, v2 = k.clone(), v.clone(), k.clone(), v.clone()
    kernels.kv_evict(k1, v1, m1, n1, 20, 4, sinks=2)
    kernels.kv_evict(k_cache=k2, v_cache=v2, mass=m2, kv_len=n2, budget=np.int64(20), recent=np.int64(4), sinks=np.int32(2))
    assert torch.equal(k1, k2) and torch.equal(v1, v2) and torch.equal(m1, m2) and torch.equal(n1, n2)
    with pytest.raises(TypeError):
        kernels.decode_sdpa(keys=k, values=v, scale=0.125)
