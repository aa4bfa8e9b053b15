"""Latent attention over a paged cache: page plans, row stores, the absorbed
and the expanded form, against plain 64-bit implementations.

Tolerances of the attention results (u = eps / 2 of the element type, the
largest relative error of one rounding): the result is rounded once (u |o|);
each softmax weight may be rounded once to the element type before it meets
its value (u sum p |v|); a score s = scale q . k in FP32 is off by at most
e = (d + 2) 2^-23 scale sum |q k| (d products, an addition that may truncate,
two scalings), which changes a weight and the sum by a factor within e^(+-e)
each, together 2 e sum p |v| (e < 0.01, doubled to cover the second order);
exp2 and the remaining FP32 steps stay below 2^-18 sum p |v| (2^-22 for the
exponential of an argument of up to 2^5, and a sum of n weights in 8 or more
partial sums).  FP16 weights below 2^-14 keep an absolute step of 2^-24: half
of it per key, where the largest weight is held as 1 or more; the result's own
smallest step likewise.  Log-sums: e, the sum's error and one FP32 rounding."""

import math

import numpy as np
import pytest
import torch

R, r = 512, 64


# --- 64-bit forms ----------------------------------------------------------


def plan64(cached, new, table, free, count, page, tokens):
    table = [list(row) for row in table]
    free = list(free[:count])
    slots, positions, starts, lens = [], [], [0], []
    for i, (c, n) in enumerate(zip(cached, new)):
        held, want = -(-c // page), -(-(c + n) // page)
        for k in range(held, want):
            table[i][k] = free.pop()
        for p in range(c, c + n):
            slots.append(table[i][p // page] * page + p % page)
            positions.append(p)
        starts.append(starts[-1] + n)
        lens.append(c + n)
    pad = tokens - len(slots)
    return table, slots + [-1] * pad, positions + [0] * pad, starts, lens, len(free)


def attend64(q, k, v, visible, scale, dtype):
    """(out, lse, tolerance, lse tolerance) of one head: q [n, d], k [m, d], v [m, dv], visible [n] keys each."""
    u = torch.finfo(dtype).eps / 2
    q, k, v = q.double(), k.double(), v.double()
    n, m = q.shape[0], k.shape[0]
    if m == 0:
        z = torch.zeros((n, v.shape[1]), dtype=torch.float64, device=q.device)
        return z, torch.full((n,), -math.inf, dtype=torch.float64, device=q.device), z, z[:, 0]
    seen = torch.arange(m, device=q.device)[None, :] < visible[:, None]
    # what is masked does not enter, whatever it holds
    s = torch.empty((n, m), dtype=torch.float64, device=q.device)
    vz = torch.where(torch.isfinite(v), v, torch.zeros_like(v))
    kz = torch.where(torch.isfinite(k), k, torch.zeros_like(k))
    s = torch.where(seen, (q @ kz.T) * scale, torch.full_like(s, -math.inf))
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - torch.where(lse.isinf(), torch.zeros_like(lse), lse)[:, None])
    out = p @ vz
    mass = p @ vz.abs()
    e = ((q.abs() @ kz.abs().T) * abs(scale) * seen).amax(-1) * (q.shape[1] + 2) * 2.0 ** -23
    tol = u * out.abs() + (u + 4 * e[:, None] + 2.0 ** -18) * mass * (1 + u) + 1e-30
    if dtype == torch.float16:
        tol = tol + m * 2.0 ** -25 * vz.abs().amax() * p.amax(-1, keepdim=True) + 2.0 ** -25
    return out, lse, tol, 2 * e + 2.0 ** -18 + lse.abs().nan_to_num(posinf=0) * 2.0 ** -22


def check(got, lse, out64, lse64, tol, lse_tol):
    err = (got.double() - out64).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{int(bad.sum())} values off, worst {float((err / tol).nan_to_num(nan=1e9).max()):.3f} x tolerance"
    if lse is not None:
        empty = lse64 == -math.inf
        assert torch.equal(lse.double() == -math.inf, empty)
        assert ((lse.double() - lse64).abs()[~empty] <= lse_tol[~empty]).all()


# --- refusals (no device) --------------------------------------------------


def lib():
    from glm53_flash_mlx_b200 import _native as N

    return N.load_library()


ONE = 16  # a pointer that is only checked


def plan_args(**kw):
    a = dict(cached=ONE, new=ONE, B=2, table=ONE, stride=4, width=4, free=ONE, cap=8, count=ONE, page=16, tokens=4,
             slots=ONE, pos=ONE, starts=ONE, lens=ONE, out=2 * ONE, status=None, host=None, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("bad", [dict(B=-1), dict(B=8193), dict(page=0), dict(width=5), dict(width=1 << 30, stride=1 << 30),
                                 dict(tokens=-1), dict(tokens=1 << 31), dict(cap=-1), dict(out=ONE), dict(starts=None),
                                 dict(slots=None), dict(free=None), dict(table=None)])
def test_plan_refuses(bad):
    assert lib().glm53_plan_pages(*plan_args(**bad)) == 1


def write_args(**kw):
    a = dict(kv=ONE, T=2, stride=576, R=512, r=64, dtype=0, w=ONE, eps=1e-6, pos=ONE, freq=ONE, inter=0, slots=ONE,
             cache=ONE, rows=64, q=ONE, heads=4, qt=256, qh=64, qo=ONE, status=None, host=None, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("bad", [dict(dtype=2), dict(T=-1), dict(R=12), dict(R=1032), dict(r=8), dict(r=272),
                                 dict(stride=568), dict(stride=580), dict(pos=None), dict(freq=None),
                                 dict(r=0, stride=512), dict(heads=0), dict(qh=63), dict(qt=4), dict(qo=None),
                                 dict(pos=None, freq=None), dict(kv=8), dict(cache=24), dict(slots=None), dict(rows=-1)])
def test_write_refuses(bad):
    assert lib().glm53_latent_cache_write(*write_args(**bad)) == 1


def absorbed_args(**kw):
    a = dict(ql=ONE, qlt=512, qlh=512, qr=ONE, qrt=64, qrh=64, T=2, H=1, R=512, r=64, dtype=0, cache=ONE, pages=4,
             page=16, table=ONE, stride=4, width=4, lens=ONE, B=2, starts=None, scale=1.0, out=ONE, lse=None, tail=0,
             ws=ONE, wsb=1 << 40, status=None, host=None, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("bad", [dict(dtype=-1), dict(R=64), dict(R=520), dict(R=640), dict(r=32), dict(H=0), dict(H=1025),
                                 dict(T=-1), dict(T=3), dict(page=4), dict(page=12), dict(pages=1 << 28),
                                 dict(width=5), dict(qlt=511), dict(qlh=504), dict(qrh=32), dict(scale=math.inf),
                                 dict(scale=math.nan), dict(ql=None), dict(qr=None), dict(out=8), dict(cache=None),
                                 dict(lens=None), dict(ws=None), dict(wsb=1)])
def test_absorbed_refuses(bad):
    assert lib().glm53_latent_absorbed(*absorbed_args(**bad)) == 1


def expanded_args(**kw):
    a = dict(qn=ONE, qnt=192, qnh=192, qr=ONE, qrt=64, qrh=64, kn=ONE, knt=192, knh=192, kr=ONE, krt=64, v=ONE, vt=256,
             vh=256, Tq=2, Tk=2, H=1, dn=192, dr=64, dv=256, dtype=0, qs=ONE, ks=ONE, B=1, scale=1.0, causal=1, out=ONE,
             lse=None, tail=0, status=None, host=None, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("bad", [dict(dtype=3), dict(dn=0), dict(dn=96), dict(dn=256), dict(dr=16), dict(dv=32), dict(dv=320),
                                 dict(Tq=-1), dict(Tk=-1), dict(H=0), dict(B=-1), dict(B=70000), dict(scale=math.nan),
                                 dict(qnt=1), dict(knh=4), dict(vt=-8), dict(qn=None), dict(kr=None), dict(v=8),
                                 dict(qs=None)])
def test_expanded_refuses(bad):
    assert lib().glm53_latent_expanded(*expanded_args(**bad)) == 1


@pytest.mark.parametrize("entry,make,bads", [
    (0, plan_args, [dict(B=-1), dict(page=0), dict(out=ONE)]),
    (1, write_args, [dict(dtype=2), dict(R=12), dict(kv=8), dict(qo=None)]),
    (2, absorbed_args, [dict(T=3), dict(scale=math.nan), dict(wsb=1), dict(width=5)]),
    (3, expanded_args, [dict(dv=32), dict(scale=math.inf), dict(B=70000), dict(qs=None)]),
])
def test_packed_call_refuses_alike(entry, make, bads):
    import struct

    names = ["glm53_plan_pages", "glm53_latent_cache_write", "glm53_latent_absorbed", "glm53_latent_expanded"]
    for bad in bads:
        args = make(**bad)
        rc = getattr(lib(), names[entry])(*args)
        why = lib().glm53_last_error()
        words = b"".join(struct.pack("d" if isinstance(a, float) else "q", a or 0) for a in args)
        assert lib().glm53_latent_call(entry, words) == rc == 1
        assert lib().glm53_last_error() == why
    assert lib().glm53_latent_call(9, b"\0" * 400) == 1 and lib().glm53_latent_call(entry, None) == 1


def test_python_refuses_before_the_device():
    import glm53_flash_mlx_b200 as G

    i32 = torch.int32
    lens, table, free = torch.zeros(2, dtype=i32), torch.zeros((2, 4), dtype=i32), torch.zeros(8, dtype=i32)
    one = torch.ones(1, dtype=i32)
    for args in [(lens.long(), lens, table, free, one), (lens, lens[:1], table, free, one),
                 (lens, lens, table[:1], free, one), (lens, lens, table.long(), free, one),
                 (lens, lens, table.t().contiguous().t(), free, one), (lens, lens, table[:1].expand(2, 4), free, one),
                 (lens, lens, table, free, lens)]:
        with pytest.raises(ValueError):
            G.plan_pages(*args, page_size=16, tokens=4)
    with pytest.raises(ValueError):
        G.plan_pages(lens, lens, table, free, one, page_size=0, tokens=4)
    kv, cache = torch.zeros((2, 576), dtype=torch.bfloat16), torch.zeros((4, 16, 576), dtype=torch.bfloat16)
    slots = torch.zeros(2, dtype=torch.int64)
    for a, kw in [((kv.float(), cache, slots), {}), ((kv, cache.half(), slots), {}), ((kv, cache[..., :512], slots), {}),
                  ((kv, cache, slots.int()), {}), ((kv, cache, slots[:1]), {}), ((kv, cache, slots), dict(rope_dim=576)),
                  ((kv, cache, slots), dict(positions=lens)), ((kv, cache, slots), dict(queries=kv[:, None, :64])),
                  ((kv, cache, slots), dict(norm_weight=kv[0, :64]))]:
        with pytest.raises(ValueError):
            G.latent_cache_write(*a, **kw)
    q, qr = torch.zeros((2, 4, 512), dtype=torch.bfloat16), torch.zeros((2, 4, 64), dtype=torch.bfloat16)
    for a, kw in [((q.float(), qr, cache, table, lens), {}), ((q, qr.half(), cache, table, lens), {}),
                  ((q[..., :500], qr, cache, table, lens), {}), ((q, None, cache, table, lens), {}),
                  ((q, qr, cache[:, :12], table, lens), {}), ((q[:1], qr[:1], cache, table, lens), {}),
                  ((q, qr, cache, table.long(), lens), {}), ((q, qr, cache, table, lens), dict(query_starts=lens)),
                  ((q, qr, cache, table[:1], lens), {})]:
        with pytest.raises(ValueError):
            G.latent_attention_absorbed(*a, scale=1.0, **kw)
    kn, kr, v = q[..., :192], kv[:, :64], q[..., :256]
    for a in [(kn.float(), qr, kn, kr, v, one, one), (kn, qr, kn, None, v, one, one), (kn, qr, kn[:1], kr, v, one, one),
              (q[..., :256], qr, q[..., :256], kr, v, one, one), (kn, qr, kn, kr, q[..., :96], one, one),
              (kn, qr, kn, kr, v, one, lens), (kn, qr, kn, kr, v, one.long(), one)]:
        with pytest.raises(ValueError):
            G.latent_attention_expanded(*a, scale=1.0)
    if not torch.cuda.is_available():
        with pytest.raises(RuntimeError, match="CUDA"):
            G.plan_pages(lens, lens, table, free, one, page_size=16, tokens=4)


# --- plan_pages ------------------------------------------------------------


def make_plan_case(B, page, most, seed):
    rng = np.random.default_rng(seed)
    cached = rng.integers(0, most + 1, B)
    new = rng.integers(0, most + 1, B)
    width = int(-(-(2 * most) // page)) + 1
    ids = rng.permutation(B * width + 7).astype(np.int32)
    table = np.full((B, width), -1, np.int32)
    n = 0
    for i in range(B):
        held = -(-int(cached[i]) // page)
        table[i, :held] = ids[n:n + held]
        n += held
    return cached.tolist(), new.tolist(), table, ids[n:]


def run_plan(cached, new, table, free, count, page, tokens, stride=None):
    import glm53_flash_mlx_b200 as G

    dev = "cuda"
    i32 = torch.int32
    B, width = table.shape
    full = torch.full((B, stride or width), -7, dtype=i32, device=dev)
    view = full[:, :width]
    view.copy_(torch.from_numpy(table))
    plan = G.plan_pages(torch.tensor(cached, dtype=i32, device=dev), torch.tensor(new, dtype=i32, device=dev), view,
                        torch.from_numpy(np.asarray(free, np.int32)).to(dev), torch.tensor([count], dtype=i32, device=dev),
                        page_size=page, tokens=tokens)
    return plan, view, full


@pytest.mark.gpu
@pytest.mark.parametrize("B,page,most,pad,stride", [(1, 16, 40, 0, None), (3, 1, 5, 4, 40), (7, 64, 200, 0, None),
                                                    (300, 16, 90, 11, None), (8192, 32, 3, 1, None), (33, 48, 700, 0, 90)])
def test_plan_matches(B, page, most, pad, stride):
    cached, new, table, free = make_plan_case(B, page, most, B + page)
    total = sum(new) + pad
    want = plan64(cached, new, table, free, len(free), page, total)
    plan, view, full = run_plan(cached, new, table, free, len(free), page, total, stride)
    assert view.cpu().numpy().tolist() == [list(map(int, row)) for row in want[0]]
    assert plan.slots.tolist() == list(map(int, want[1]))
    assert plan.positions.tolist() == want[2]
    assert plan.query_starts.tolist() == want[3]
    assert plan.seq_lens.tolist() == want[4]
    assert plan.free_count.tolist() == [want[5]]
    if stride:
        assert (full[:, table.shape[1]:] == -7).all()  # what lies behind the rows is left as it was


@pytest.mark.gpu
def test_plan_of_nothing():
    plan, _, _ = run_plan([], [], np.zeros((0, 4), np.int32), [1, 2], 2, 16, 3)
    assert plan.slots.tolist() == [-1] * 3 and plan.query_starts.tolist() == [0] and plan.free_count.tolist() == [2]
    plan, _, _ = run_plan([5, 0], [0, 0], np.array([[3], [-1]], np.int32), [1], 1, 16, 0)
    assert plan.seq_lens.tolist() == [5, 0] and plan.free_count.tolist() == [1]


@pytest.mark.gpu
@pytest.mark.parametrize("case", ["pages", "tokens", "width", "negative", "count"])
def test_plan_that_does_not_fit_plans_nothing(case):
    import glm53_flash_mlx_b200 as G

    cached, new, table, free = make_plan_case(9, 16, 60, 5)
    new[4] = 60
    count, tokens = len(free), sum(new)
    if case == "pages":
        count = 2
    elif case == "tokens":
        tokens -= 1
    elif case == "width":
        new[3] = 16 * table.shape[1] - cached[3] + 1
        tokens = sum(new)
    elif case == "negative":
        new[2] = -1
    else:
        count = len(free) + 1
    plan, view, _ = run_plan(cached, new, table, free, count, 16, tokens)
    with pytest.raises(RuntimeError, match="page plan"):
        G.check_latent_status()
    assert np.array_equal(view.cpu().numpy(), table)
    assert (plan.slots == -1).all() and (plan.positions == 0).all() and (plan.query_starts == 0).all()
    assert plan.seq_lens.tolist() == cached and plan.free_count.tolist() == [count]
    G.check_latent_status()  # raised once


# --- latent_cache_write ----------------------------------------------------


def write64(kv, slots, w, pos, freq, interleaved, eps, latent):
    x = kv.double().clone()
    if w is not None:
        x[:, :latent] = x[:, :latent] / (x[:, :latent].pow(2).mean(-1, keepdim=True) + eps).sqrt() * w.double()
    if pos is not None:
        x[:, latent:] = turn64(x[:, latent:], pos, freq, interleaved)
    return x


def turn64(x, pos, freq, interleaved):
    x = x.double()
    ang = pos.double().view(-1, *[1] * (x.dim() - 1)) * freq
    c, s = ang.cos(), ang.sin()
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    a, b = x.chunk(2, -1)
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def rounded_close(got, want, scale):
    """One rounding of the result, and FP32 steps relative to the values that were combined."""
    fi = torch.finfo(got.dtype)
    tol = fi.eps / 2 * want.abs() * (1 + 2.0 ** -10) + 2.0 ** -19 * scale + fi.tiny * fi.eps / 2
    err = (got.double() - want).abs()
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,latent,rope,heads,norm,interleaved,page", [
    (1, 512, 64, 64, True, False, 64), (9, 512, 64, 5, True, True, 16), (130, 512, 64, 0, True, False, 48),
    (17, 8, 16, 1, True, False, 3), (33, 1024, 256, 3, False, True, 16), (8, 512, 0, 0, True, False, 16),
    (5, 256, 64, 0, False, False, 16), (1000, 512, 64, 64, True, False, 64), (1111, 128, 128, 9, True, True, 16)])
def test_write_matches(dtype, T, latent, rope, heads, norm, interleaved, page):
    import glm53_flash_mlx_b200 as G

    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(T + latent)
    pages = -(-T // page) + 2
    wide = torch.randn((T, latent + rope + 8), generator=g, device=dev).to(dtype)
    kv = wide[:, :latent + rope]  # strided rows
    cache = torch.randn((pages, page, latent + rope), generator=g, device=dev).to(dtype)
    before = cache.clone()
    slots = torch.randperm(pages * page, generator=g, device=dev)[:T]
    if T > 4:
        slots[T // 2] = -1
    w = (1 + 0.2 * torch.randn(latent, generator=g, device=dev)).to(dtype) if norm else None
    pos = freq = q = None
    if rope:
        pos = torch.randint(0, 1 << 20, (T,), generator=g, device=dev, dtype=torch.int32)
        freq = 10000.0 ** (-torch.arange(0, rope, 2, device=dev, dtype=torch.float64) / rope)
        if heads:
            q = torch.randn((T, heads, rope + 24), generator=g, device=dev).to(dtype)[..., 8:8 + rope]
    got = G.latent_cache_write(kv, cache, slots, rope_dim=rope, norm_weight=w, eps=1e-5, positions=pos, inv_freq=freq,
                               interleaved=interleaved, queries=q)
    G.check_latent_status()
    want = write64(kv, slots, w, pos, freq, interleaved, 1e-5, latent)
    flat, old = cache.view(-1, latent + rope), before.view(-1, latent + rope)
    stored = slots[slots >= 0]
    rounded_close(flat[stored], want[slots >= 0], 8.0)
    kept = torch.ones(pages * page, dtype=torch.bool, device=dev)
    kept[stored] = False
    assert torch.equal(flat[kept], old[kept])
    if heads:
        rounded_close(got, turn64(q, pos, freq, interleaved), 8.0)
    else:
        assert got is None


@pytest.mark.gpu
def test_write_reports_a_slot_outside_the_cache():
    import glm53_flash_mlx_b200 as G

    kv = torch.ones((3, 576), dtype=torch.bfloat16, device="cuda")
    cache = torch.zeros((2, 16, 576), dtype=torch.bfloat16, device="cuda")
    G.latent_cache_write(kv, cache, torch.tensor([1, 32, 1 << 40], device="cuda"))
    with pytest.raises(IndexError, match="slot"):
        G.check_latent_status()
    assert (cache.view(32, 576)[1] == 1).all() and cache.float().sum() == 576


@pytest.mark.gpu
def test_write_reads_overlapping_rows():
    import glm53_flash_mlx_b200 as G

    run = torch.randn(576 + 8 * 4, device="cuda").to(torch.bfloat16)
    kv = run.unfold(0, 576, 8)  # five rows, each eight values behind the last
    cache = torch.zeros((1, 16, 576), dtype=torch.bfloat16, device="cuda")
    G.latent_cache_write(kv, cache, torch.arange(5, device="cuda"))
    G.check_latent_status()
    assert torch.equal(cache[0, :5], kv)


@pytest.mark.gpu
def test_write_refuses_rows_of_the_cache():
    import glm53_flash_mlx_b200 as G

    cache = torch.zeros((4, 16, 576), dtype=torch.bfloat16, device="cuda")
    slots, pos = torch.arange(3, device="cuda"), torch.arange(3, dtype=torch.int32, device="cuda")
    freq = torch.ones(32, dtype=torch.float64, device="cuda")
    rows = cache.view(64, 576)
    for at in (0, 61):
        with pytest.raises(ValueError, match="outside the cache"):
            G.latent_cache_write(rows[at:at + 3], cache, slots)
        with pytest.raises(ValueError, match="outside the cache"):
            G.latent_cache_write(torch.ones_like(rows[:3]), cache, slots, positions=pos, inv_freq=freq,
                                 queries=rows[at:at + 3, 512:].unsqueeze(1))
    # the rows beside a cache that is a part of a larger buffer are not in it
    G.latent_cache_write(rows[45:48], cache[3:], slots)
    G.latent_cache_write(rows[16:19], cache[:1], slots)
    G.latent_cache_write(rows[48:48], cache, slots[:0])
    G.check_latent_status()


@pytest.mark.gpu
def test_write_reads_queries_that_overlap():
    import glm53_flash_mlx_b200 as G

    dev, dt = "cuda", torch.bfloat16
    run = torch.randn(1000, device=dev).to(dt)
    pos = torch.arange(3, dtype=torch.int32, device=dev)
    freq = torch.rand(32, dtype=torch.float64, device=dev)
    for strides in ((200, 8, 1), (0, 64, 1), (200, 0, 1), (8, 16, 1), (7, 5, 1), (200, 64, 2)):
        q = run.as_strided((3, 5, 64), strides)
        cache = torch.zeros((1, 16, 576), dtype=dt, device=dev)
        got = G.latent_cache_write(torch.ones((3, 576), dtype=dt, device=dev), cache, torch.arange(3, device=dev),
                                   positions=pos, inv_freq=freq, queries=q)
        G.check_latent_status()
        rounded_close(got, turn64(q, pos, freq, False), 8.0)


@pytest.mark.gpu
def test_write_of_one_slot_twice_leaves_the_other_rows():
    """What a row holds that two tokens name is not defined; equal tokens give their row, and all other rows are right."""
    import glm53_flash_mlx_b200 as G

    kv = torch.randn((300, 576), device="cuda").to(torch.bfloat16)
    kv[200:250] = kv[100:150]
    slots = torch.randperm(400, device="cuda")[:300]
    slots[200:250] = slots[100:150]  # the same rows twice
    slots[250:300] = slots[0]        # different rows in one slot
    cache = torch.full((25, 16, 576), 5.0, dtype=torch.bfloat16, device="cuda")
    G.latent_cache_write(kv, cache, slots)
    G.check_latent_status()
    want = torch.full((400, 576), 5.0, dtype=torch.bfloat16, device="cuda")
    want[slots[1:200]] = kv[1:200]
    rest = torch.arange(400, device="cuda") != slots[0]
    assert torch.equal(cache.view(400, 576)[rest], want[rest])


# --- absorbed form ---------------------------------------------------------


def make_absorbed(lens, queries, H, latent, rope, page, dtype, seed=0, strided=False):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    B = len(lens)
    width = max(1, max(-(-n // page) for n in lens))
    pages = B * width + 3
    # pages that no request holds, and rows behind a request's end, hold NaN and infinities
    cache = torch.full((pages, page, latent + rope), float("nan"), dtype=dtype, device=dev)
    cache[:, 1::2] = float("inf")
    table = torch.full((B, width + 2), -1, dtype=torch.int32, device=dev)
    ids = torch.randperm(pages, generator=g, device=dev)
    rows = []
    for i, n in enumerate(lens):
        held = -(-n // page)
        own = ids[i * width:i * width + held]
        table[i, :held] = own.int()
        x = torch.randn((n, latent + rope), generator=g, device=dev).to(dtype)
        at = torch.arange(n, device=dev)
        if n:
            cache.view(-1, latent + rope)[own[at // page] * page + at % page] = x
        rows.append(x)
    T = sum(queries)
    if strided:
        q = torch.randn((T, H, latent + rope + 8), generator=g, device=dev).to(dtype)
        ql, qr = q[..., :latent], q[..., latent:latent + rope]
    else:
        ql = torch.randn((T, H, latent), generator=g, device=dev).to(dtype)
        qr = torch.randn((T, H, rope), generator=g, device=dev).to(dtype)
    starts = torch.tensor(np.concatenate([[0], np.cumsum(queries)]), dtype=torch.int32, device=dev)
    return ql, (qr if rope else None), cache, table, torch.tensor(lens, dtype=torch.int32, device=dev), starts, rows


def absorbed64(ql, qr, rows, lens, queries, scale, dtype):
    T, H, latent = ql.shape
    out, lse = torch.zeros((T, H, latent), dtype=torch.float64, device=ql.device), None
    tol = torch.zeros_like(out)
    lse = torch.zeros((T, H), dtype=torch.float64, device=ql.device)
    ltol = torch.zeros_like(lse)
    t = 0
    for n, nq, x in zip(lens, queries, rows):
        for j in range(nq):
            seen = max(0, n - (nq - 1 - j))
            q = ql[t] if qr is None else torch.cat([ql[t], qr[t]], -1)
            vis = torch.full((H,), seen, device=ql.device)
            out[t], lse[t], tol[t], ltol[t] = attend64(q, x[:seen], x[:seen, :latent], vis, scale, dtype)
            t += 1
    return out, lse, tol, ltol


ABSORBED = [
    # lens, queries, heads, latent, rope, page, strided
    ([777], [1], 64, 512, 64, 64, False),
    ([1], [1], 64, 512, 64, 16, False),
    ([0, 5, 0], [1, 1, 1], 64, 512, 64, 16, False),
    ([63, 64, 65, 127, 128, 129], [1] * 6, 64, 512, 64, 64, True),
    ([300, 17, 0, 2], [2, 3, 2, 4], 16, 512, 64, 16, False),
    ([40, 1000], [0, 5], 5, 512, 64, 8, True),
    ([500, 33], [1, 1], 1, 128, 64, 48, False),
    ([500, 33], [1, 1], 65, 256, 0, 128, False),
    ([200], [1], 130, 384, 64, 32, False),
    ([9000], [1], 64, 512, 64, 64, False),
    ([2500] * 3 + [1, 0, 70], [1] * 6, 32, 512, 0, 16, False),
    (list(range(0, 400)), [1] * 400, 8, 128, 64, 16, False),
    ([300, 20, 90], [300, 1, 70], 4, 128, 64, 32, False),   # a prompt's worth of tokens in one request
    ([50, 700], [80, 65], 70, 128, 0, 16, True),            # more tokens than rows; two groups of heads
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", range(len(ABSORBED)))
def test_absorbed_matches(dtype, case):
    import glm53_flash_mlx_b200 as G

    lens, queries, H, latent, rope, page, strided = ABSORBED[case]
    ql, qr, cache, table, n, starts, rows = make_absorbed(lens, queries, H, latent, rope, page, dtype, case, strided)
    scale = (latent + rope) ** -0.5 * 1.5
    one_each = all(q == 1 for q in queries)
    out, lse = G.latent_attention_absorbed(ql, qr, cache, table, n, scale=scale,
                                           query_starts=None if one_each else starts, return_lse=True)
    G.check_latent_status()
    check(out, lse, *absorbed64(ql, qr, rows, lens, queries, scale, dtype))
    again = G.latent_attention_absorbed(ql, qr, cache, table, n, scale=scale, query_starts=starts)
    assert torch.equal(again, out)  # same bits from call to call, with and without lse


@pytest.mark.gpu
def test_absorbed_scores_that_grow():
    """Scores that rise along the keys, so that the running maximum is replaced again and again, and a
    negative scale."""
    import glm53_flash_mlx_b200 as G

    lens, queries, H = [1500, 700], [1, 1], 64
    for sign in (1.0, -1.0):
        ql, qr, cache, table, n, starts, rows = make_absorbed(lens, queries, H, 512, 64, 64, torch.bfloat16, 3)
        ql.fill_(0.25)
        for i, m in enumerate(lens):
            ramp = (torch.arange(m, device="cuda") / m * 4).to(torch.bfloat16)
            rows[i][:, :128] = ramp[:, None] * sign
            at = torch.arange(m, device="cuda")
            cache.view(-1, 576)[table[i].long()[at // 64] * 64 + at % 64] = rows[i]
        out, lse = G.latent_attention_absorbed(ql, qr, cache, table, n, scale=0.5 * sign, return_lse=True)
        check(out, lse, *absorbed64(ql, qr, rows, lens, queries, 0.5 * sign, torch.bfloat16))


@pytest.mark.gpu
def test_absorbed_padded_batch_keeps_or_zeroes_the_rest():
    import glm53_flash_mlx_b200 as G

    lens, queries = [100, 30], [2, 1]
    ql, qr, cache, table, n, starts, rows = make_absorbed(lens, queries, 16, 512, 64, 16, torch.bfloat16, 9)
    pad = lambda x: torch.cat([x, torch.full((4, *x.shape[1:]), float("nan"), dtype=x.dtype, device="cuda")])
    new, lse = G.latent_attention_absorbed(pad(ql), pad(qr), cache, table, n, scale=0.05, query_starts=starts,
                                           return_lse=True)
    want = G.latent_attention_absorbed(ql, qr, cache, table, n, scale=0.05, query_starts=starts)
    assert torch.equal(new[:3], want) and (new[3:] == 0).all() and (lse[3:] == -math.inf).all()
    given = torch.full_like(new, 7.0)
    got = G.latent_attention_absorbed(pad(ql), pad(qr), cache, table, n, scale=0.05, query_starts=starts, out=given)
    assert got is given and torch.equal(given[:3], want) and (given[3:] == 7).all()
    G.check_latent_status()


def stale(*shape):
    """Leaves blocks of this size that hold other values to the allocator."""
    blocks = [torch.full(shape, 7.0, device="cuda") for _ in range(8)]
    del blocks


@pytest.mark.gpu
def test_absorbed_log_sums_behind_the_last_token_of_a_given_result():
    import glm53_flash_mlx_b200 as G

    lens, queries = [100, 30, 5], [2, 1, 0]
    ql, qr, cache, table, n, starts, _ = make_absorbed(lens, queries, 16, 512, 64, 16, torch.bfloat16, 9)
    ql, qr = (torch.cat([x, x[:2], x[:2]]) for x in (ql, qr))
    for starts in (starts, starts + 2):  # four tokens behind the last request; two before the first and behind the last
        first = int(starts[0])
        want, lse = G.latent_attention_absorbed(ql, qr, cache, table, n, scale=0.05, query_starts=starts, return_lse=True)
        given = torch.full_like(want, 7.0)
        stale(7, 16)
        got, again = G.latent_attention_absorbed(ql, qr, cache, table, n, scale=0.05, query_starts=starts, out=given,
                                                 return_lse=True)
        outside = torch.ones(7, dtype=torch.bool, device="cuda")
        outside[first:first + 3] = False
        assert (again[outside] == -math.inf).all() and torch.equal(again, lse)
        assert (given[outside] == 7).all() and torch.equal(given[~outside], want[~outside])
    G.check_latent_status()


@pytest.mark.gpu
def test_outputs_that_overlap_inputs_are_refused():
    import glm53_flash_mlx_b200 as G

    ql, qr, cache, table, n, _, _ = make_absorbed([100, 30], [1, 1], 16, 512, 64, 16, torch.bfloat16, 9)
    with pytest.raises(ValueError, match="overlap"):
        G.latent_attention_absorbed(ql, qr, cache, table, n, scale=0.05, out=ql)
    t = make_expanded([40], [40], 2, 128, 64, 128, torch.bfloat16, 8)
    with pytest.raises(ValueError, match="overlap"):
        v = t[4].contiguous()
        G.latent_attention_expanded(*t[:4], v, *t[5:], scale=0.07, out=v)


@pytest.mark.gpu
def test_absorbed_reports_bad_pages_and_lengths():
    import glm53_flash_mlx_b200 as G

    lens = [100, 30]
    ql, qr, cache, table, n, starts, rows = make_absorbed(lens, [1, 1], 16, 512, 64, 16, torch.bfloat16, 9)
    want = G.latent_attention_absorbed(ql, qr, cache, table, n, scale=0.05)
    for bad in (-1, cache.shape[0], 2 ** 31 - 1, -2 ** 31):
        t2 = table.clone()
        t2[1, 1] = bad
        got = G.latent_attention_absorbed(ql, qr, cache, t2, n, scale=0.05)
        with pytest.raises(IndexError, match="page"):
            G.check_latent_status()
        assert torch.equal(got[0], want[0])  # the other request is not touched by it
    for bad in (-1, 16 * table.shape[1] + 1):
        n2 = n.clone()
        n2[1] = bad
        got = G.latent_attention_absorbed(ql, qr, cache, table, n2, scale=0.05)
        with pytest.raises(RuntimeError):
            G.check_latent_status()
        assert torch.equal(got[0], want[0]) and (got[1] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("starts", [[0, 40, 0, 40, 0, 40], [0, 10, 50, 30, 35, 40], [-1, 1, 2, 3, 4, 5],
                                    [0, 10, 20, 30, 40, 41], [40, 30, 20, 10, 5, 0]])
def test_absorbed_starts_out_of_order_bound_no_token(starts):
    import glm53_flash_mlx_b200 as G

    lens = [3000, 100, 2000, 40, 500]
    ql, qr, cache, table, n, _, _ = make_absorbed(lens, [8] * 5, 16, 512, 64, 16, torch.bfloat16, 11)
    bad = torch.tensor(starts, dtype=torch.int32, device="cuda")
    out, lse = G.latent_attention_absorbed(ql, qr, cache, table, n, scale=0.05, query_starts=bad, return_lse=True)
    with pytest.raises(RuntimeError):
        G.check_latent_status()
    assert (out == 0).all() and (lse == -math.inf).all()
    given = torch.ones_like(out)
    G.latent_attention_absorbed(ql, qr, cache, table, n, scale=0.05, query_starts=bad, out=given)
    with pytest.raises(RuntimeError):
        G.check_latent_status()
    assert (given == 1).all()


# --- expanded form ---------------------------------------------------------


def make_expanded(nq, nk, H, dn, dr, dv, dtype, seed=0):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    Tq, Tk = sum(nq), sum(nk)
    q = torch.randn((Tq, H, dn + dr), generator=g, device=dev).to(dtype)
    kv = torch.randn((Tk, H, dn + dv), generator=g, device=dev).to(dtype)
    latent = torch.randn((Tk, 512 + dr), generator=g, device=dev).to(dtype)
    qs = torch.tensor(np.concatenate([[0], np.cumsum(nq)]), dtype=torch.int32, device=dev)
    ks = torch.tensor(np.concatenate([[0], np.cumsum(nk)]), dtype=torch.int32, device=dev)
    qr, kr = (q[..., dn:], latent[:, 512:]) if dr else (None, None)
    return q[..., :dn], qr, kv[..., :dn], kr, kv[..., dn:], qs, ks


def expanded64(qn, qr, kn, kr, v, nq, nk, scale, causal, dtype):
    Tq, H, dn = qn.shape
    dv = v.shape[2]
    out = torch.zeros((Tq, H, dv), dtype=torch.float64, device=qn.device)
    tol, lse = torch.zeros_like(out), torch.zeros((Tq, H), dtype=torch.float64, device=qn.device)
    ltol = torch.zeros_like(lse)
    qa = ka = 0
    for a, b in zip(nq, nk):
        vis = torch.arange(a, device=qn.device) + (b - a) + 1 if causal else torch.full((a,), b, device=qn.device)
        vis = vis.clamp(0, b)
        for h in range(H if a else 0):
            q, k = qn[qa:qa + a, h], kn[ka:ka + b, h]
            if qr is not None:
                q, k = torch.cat([q, qr[qa:qa + a, h]], -1), torch.cat([k, kr[ka:ka + b]], -1)
            s = slice(qa, qa + a)
            out[s, h], lse[s, h], tol[s, h], ltol[s, h] = attend64(q, k, v[ka:ka + b, h], vis, scale, dtype)
        qa, ka = qa + a, ka + b
    return out, lse, tol, ltol


EXPANDED = [
    # queries, keys, heads, nope, rope, value, causal
    ([256], [256], 4, 192, 64, 256, True),
    ([1], [1], 3, 192, 64, 256, True),
    ([1], [1000], 2, 192, 64, 256, True),
    ([129, 1, 0, 127, 128], [129, 640, 5, 300, 128], 2, 128, 64, 128, True),
    ([300], [300], 2, 64, 0, 64, True),
    ([200, 40], [500, 0], 1, 192, 64, 192, False),
    ([130, 20], [50, 7], 2, 64, 64, 256, True),   # fewer keys than queries: the first rows see none
    ([513], [1100], 1, 256, 0, 256, True),
    ([3] * 40, list(range(3, 43)), 1, 128, 64, 64, True),
    ([700], [700], 1, 192, 64, 256, False),
    ([700, 300, 1000], [701, 1300, 1000], 2, 192, 64, 256, True),
    ([400, 257], [400, 258], 3, 128, 64, 128, True),
    ([600, 300], [20, 310], 1, 64, 64, 128, True),
    ([385], [2000], 1, 128, 0, 256, False),
    ([200] * 8, [2200] * 8, 4, 192, 64, 256, True),  # three tiles that the mask cuts, loaded one behind the other
    ([250, 129], [2001, 3333], 2, 128, 64, 128, True),
    ([1], [3000], 2, 192, 64, 256, True),
    ([100, 28], [2600, 2700], 3, 192, 64, 256, True),  # one query tile a request, long keys
    ([5] * 150 + [140] + [2, 0] * 100, [9] * 150 + [150] + [2, 3] * 100, 2, 64, 64, 64, True),  # many requests
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", range(len(EXPANDED)))
def test_expanded_matches(dtype, case):
    import glm53_flash_mlx_b200 as G

    nq, nk, H, dn, dr, dv, causal = EXPANDED[case]
    t = make_expanded(nq, nk, H, dn, dr, dv, dtype, case)
    scale = (dn + dr) ** -0.5 * 1.5
    out, lse = G.latent_attention_expanded(*t, scale=scale, causal=causal, return_lse=True)
    G.check_latent_status()
    check(out, lse, *expanded64(*t[:5], nq, nk, scale, causal, dtype))
    assert torch.equal(G.latent_attention_expanded(*t, scale=scale, causal=causal), out)


@pytest.mark.gpu
def test_expanded_scores_that_grow():
    import glm53_flash_mlx_b200 as G

    for nq, sign in (([260], 1), ([100], 1), ([260], -1)):
        nk = [900]
        qn, qr, kn, kr, v, qs, ks = make_expanded(nq, nk, 2, 192, 64, 256, torch.bfloat16, 4)
        qn = torch.full_like(qn, 0.25)
        kn = kn.clone()
        kn[..., :64] = (torch.arange(900, device="cuda") / 900 * 8).to(torch.bfloat16)[:, None, None] * sign
        out, lse = G.latent_attention_expanded(qn, qr, kn, kr, v, qs, ks, scale=0.5 * sign, return_lse=True)
        check(out, lse, *expanded64(qn, qr, kn, kr, v, nq, nk, 0.5 * sign, True, torch.bfloat16))
    t = make_expanded([150], [300], 2, 128, 64, 128, torch.float16, 5)
    out, lse = G.latent_attention_expanded(*t, scale=0.0, return_lse=True)  # the mean of what each row sees
    check(out, lse, *expanded64(*t[:5], [150], [300], 0.0, True, torch.float16))


@pytest.mark.gpu
@pytest.mark.parametrize("B,nq,nk,H,at", [(100, 40, 60, 16, 90), (3, 300, 2200, 2, 1), (300, 3, 5, 4, 250)])
@pytest.mark.parametrize("which", ["queries", "keys"])
def test_expanded_reports_starts_of_any_request(B, nq, nk, H, at, which):
    """However many units come before it; the requests beside it keep their results."""
    import glm53_flash_mlx_b200 as G

    *t, qs, ks = make_expanded([nq] * B, [nk] * B, H, 128, 64, 128, torch.bfloat16, 7)
    want = G.latent_attention_expanded(*t, qs, ks, scale=0.07)
    bad = (qs if which == "queries" else ks).clone()
    bad[at + 1] = -1  # the end of request `at`, the start of the next
    out = torch.ones_like(want)
    G.latent_attention_expanded(*t, *((bad, ks) if which == "queries" else (qs, bad)), scale=0.07, out=out)
    with pytest.raises(RuntimeError):
        G.check_latent_status()
    first, last = at * nq, (at + 2) * nq
    assert torch.equal(out[:first], want[:first]) and torch.equal(out[last:], want[last:])
    if which == "keys":
        assert (out[first:last] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("what", [math.nan, math.inf])
def test_expanded_masked_keys_and_values_do_not_enter_large(what):
    """The same with more than 128 queries a request, at every place of a 256-row unit."""
    import glm53_flash_mlx_b200 as G

    nq, nk = [600, 300], [600, 333]
    qn, qr, kn, kr, v, qs, ks = make_expanded(nq, nk, 2, 192, 64, 256, torch.bfloat16, 6)
    clean = G.latent_attention_expanded(qn, qr, kn, kr, v, qs, ks, scale=0.06)
    bad, hit = v.clone(), torch.zeros_like(clean, dtype=torch.bool)
    for key, head, col in [(0, 0, 3), (130, 0, 70), (255, 1, 130), (256, 1, 0), (300, 0, 255), (511, 1, 64), (599, 0, 200)]:
        bad[key, head, col] = what
        hit[key:600, head, col] = True
    bad[600 + 332, 1, 255] = what
    hit[899, 1, 255] = True
    got = G.latent_attention_expanded(qn, qr, kn, kr, bad, qs, ks, scale=0.06)
    G.check_latent_status()
    assert torch.equal(got[~hit], clean[~hit])
    assert got[hit].isnan().all() if math.isnan(what) else (got[hit] == math.inf).all()
    kbad = kn.clone()
    kbad[600:] = math.nan  # the second request's keys
    got = G.latent_attention_expanded(qn, qr, kbad, kr, v, qs, ks, scale=0.06)
    assert torch.equal(got[:600], clean[:600]) and got[600:].isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("what", [math.nan, math.inf])
def test_expanded_masked_keys_and_values_do_not_enter(what):
    """A request's rows that are not finite stay out of the requests beside it and of the rows that do not
    see them; the rows that see them get them."""
    import glm53_flash_mlx_b200 as G

    nq, nk = [70, 100, 90], [70, 180, 90]
    qn, qr, kn, kr, v, qs, ks = make_expanded(nq, nk, 2, 192, 64, 256, torch.bfloat16, 6)
    kn, v, kr = kn.clone(), v.clone(), kr.clone()
    clean = G.latent_attention_expanded(qn, qr, kn, kr, v, qs, ks, scale=0.06)
    v[70 + 150, 0, 5] = what    # seen by queries 70.. of the second request
    v[70 + 151, 1, 200] = what
    kn[70 + 160, :, 3] = math.nan  # seen by queries 80..
    got = G.latent_attention_expanded(qn, qr, kn, kr, v, qs, ks, scale=0.06)
    G.check_latent_status()
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[70 + 70:170, 0, 5] = True
    hit[70 + 71:170, 1, 200] = True
    lost = torch.zeros_like(hit)
    lost[70 + 80:170] = True
    assert got[lost].isnan().all()
    if math.isnan(what):
        assert got[hit & ~lost].isnan().all()
    else:
        assert (got[hit & ~lost] == math.inf).all()
    assert torch.equal(got[~hit & ~lost], clean[~hit & ~lost])


@pytest.mark.gpu
def test_expanded_rows_outside_every_request():
    import glm53_flash_mlx_b200 as G

    nq, nk = [40, 30], [60, 30]
    t = make_expanded(nq, nk, 3, 128, 64, 128, torch.bfloat16, 8)
    want = G.latent_attention_expanded(*t, scale=0.07)
    more = lambda x: torch.cat([x, torch.full((5, *x.shape[1:]), math.nan, dtype=x.dtype, device="cuda")])
    q = (more(t[0]), more(t[1]))
    new, lse = G.latent_attention_expanded(*q, *t[2:], scale=0.07, return_lse=True)
    assert torch.equal(new[:70], want) and (new[70:] == 0).all() and (lse[70:] == -math.inf).all()
    given = torch.full_like(new, 3.0)
    G.latent_attention_expanded(*q, *t[2:], scale=0.07, out=given)
    assert torch.equal(given[:70], want) and (given[70:] == 3).all()
    bad = t[6].clone()
    bad[2] = 91  # past the keys
    got = G.latent_attention_expanded(*t[:6], bad, scale=0.07)
    with pytest.raises(RuntimeError):
        G.check_latent_status()
    assert torch.equal(got[:40], want[:40]) and (got[40:] == 0).all()


def rows_of_requests(starts, rows):
    """Which request each row belongs to (-1: none), whatever the starts hold."""
    owner, top = [-1] * rows, 0
    for i, (a, b) in enumerate(zip(starts, starts[1:])):
        if 0 <= a <= rows:
            top = max(top, a)
        if top <= a <= b <= rows:
            owner[a:b] = [i] * (b - a)
    return owner


OUT_OF_ORDER = [  # starts, rows
    ([0, 5, 8], 6), ([0, 50, 30], 50), ([0, 40, 0, 40], 40), ([0, 40, 0, 40, 0, 40], 40), ([0, 10, 50, 30, 35, 40], 40),
    ([-1, 1, 2, 3, 4, 5], 40), ([0, 10, 20, 30, 40, 41], 40), ([40, 30, 20, 10, 5, 0], 40), ([0, 300, 100, 310, 305, 520], 530),
    ([7, 20, 900, 15, 25, -4, 30, 300], 400), ([2 ** 31 - 1, -2 ** 31, 3, 9], 12), ([0, 2 ** 31 - 1, 0, 5], 9),
    ([0, 500, 200, 600, 1000], 1100), ([3 * (i % 40) + i // 7 for i in range(260)], 150)]


def test_rows_of_requests():
    assert rows_of_requests([0, 2, 2, 5], 6) == [0, 0, 2, 2, 2, -1]
    assert rows_of_requests([0, 5, 8], 6) == [0] * 5 + [-1]
    assert rows_of_requests([0, 4, 0, 4], 4) == [0] * 4
    assert rows_of_requests([3, 9, 1, 4, 6], 8) == [-1] * 3 + [2] * 0 + [-1] + [3] * 2 + [-1] * 2


@pytest.mark.gpu
@pytest.mark.parametrize("case,keys,H", [(c, k, 2) for c in range(len(OUT_OF_ORDER)) for k in (30, 300, 2300)] +
                         [(0, 4000, 64), (2, 4000, 64)])
def test_expanded_starts_out_of_order(case, keys, H):
    """Every row is written by one request or counts as a row outside every request, with CTAs that walk, that take a
    unit each and that work in pairs."""
    import glm53_flash_mlx_b200 as G

    starts, rows = OUT_OF_ORDER[case]
    B, i32 = len(starts) - 1, torch.int32
    if B > 100:
        keys //= 10
    qn, qr, kn, kr, v, _, ks = make_expanded([rows] + [0] * (B - 1), [keys] * B, H, 128, 64, 128, torch.bfloat16, case)
    bad = torch.tensor(starts, dtype=torch.int64).to(i32).cuda()
    owner = torch.tensor(rows_of_requests(starts, rows), device="cuda")
    stale(rows, H)
    out, lse = G.latent_attention_expanded(qn, qr, kn, kr, v, bad, ks, scale=0.07, return_lse=True)
    with pytest.raises(RuntimeError):
        G.check_latent_status()
    none = owner < 0
    assert (out[none] == 0).all() and (lse[none] == -math.inf).all()
    kept = sorted(set(owner[~none].tolist()))
    # the same requests in order, their rows gathered; each keeps its own keys
    own = [int((owner == i).sum()) for i in kept]
    if kept:
        take = lambda x: x[~none]
        got = expanded64(take(qn), take(qr), *(torch.cat([x[i * keys:(i + 1) * keys] for i in kept]) for x in (kn, kr, v)),
                         own, [keys] * len(kept), 0.07, True, torch.bfloat16)
        check(out[~none], lse[~none], *got)
    given = torch.full_like(out, 3.0)
    _, again = G.latent_attention_expanded(qn, qr, kn, kr, v, bad, ks, scale=0.07, out=given, return_lse=True)
    with pytest.raises(RuntimeError):
        G.check_latent_status()
    assert (given[none] == 3).all() and torch.equal(given[~none], out[~none]) and torch.equal(again, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("nk", [[60, 30], [4500, 30]])  # CTAs alone, CTA pairs
def test_expanded_log_sums_behind_the_last_query_of_a_given_result(nk):
    import glm53_flash_mlx_b200 as G

    nq = [240, 30]
    *t, qs, ks = make_expanded(nq, nk, 3, 128, 64, 128, torch.bfloat16, 8)
    t[0], t[1] = (torch.cat([x, x[:5]]) for x in t[:2])
    for qs in (qs, qs + 2):  # five queries behind the last request; two before the first and three behind the last
        first = int(qs[0])
        want, lse = G.latent_attention_expanded(*t, qs, ks, scale=0.07, return_lse=True)
        given = torch.full_like(want, 7.0)
        stale(275, 3)
        got, again = G.latent_attention_expanded(*t, qs, ks, scale=0.07, out=given, return_lse=True)
        outside = torch.ones(275, dtype=torch.bool, device="cuda")
        outside[first:first + 270] = False
        assert (again[outside] == -math.inf).all() and torch.equal(again, lse)
        assert (given[outside] == 7).all() and torch.equal(given[~outside], want[~outside])
    G.check_latent_status()


@pytest.mark.gpu
@pytest.mark.parametrize("nq", [1, 130, 200])
@pytest.mark.parametrize("nats", [17.5, 16.0, 14.0])
def test_expanded_sums_many_small_weights(nats, nq):
    """One key far above 30,000 others, which together make up to 2% of the sum.  The log-sum's error: a tile's 32
    additions and those of 235 tiles, half a step of 2^-23 each, 1.6e-5; the score's and the exponential's steps, 2^-18;
    one rounding."""
    import glm53_flash_mlx_b200 as G

    n, dt = 30000, torch.bfloat16
    k = torch.zeros((n, 2, 64), dtype=dt, device="cuda")
    k[0, :, 0] = nats
    q = torch.zeros((nq, 2, 64), dtype=dt, device="cuda")
    q[..., 0] = 1
    starts = [torch.tensor([0, m], dtype=torch.int32, device="cuda") for m in (nq, n)]
    for dv in (64, 128):  # CTAs alone, CTA pairs
        v = torch.zeros((n, 2, dv), dtype=dt, device="cuda")
        _, lse = G.latent_attention_expanded(q, None, k, None, v, *starts, scale=1.0, causal=False, return_lse=True)
        G.check_latent_status()
        want = nats + math.log1p((n - 1) * math.exp(-nats))
        assert ((lse.double() - want).abs() <= 1.6e-5 + 2.0 ** -18 + want * 2.0 ** -24).all(), float((lse - want).abs().max())


# --- weights far below the largest -----------------------------------------


def small_weights(n, nats, width, dtype):
    """n keys of `width` values: the first scores `nats` above all others (q = 1 in the first place, scale 1) and has
    the values 0, the others 1 in places 8 and up; and what softmax gives there, with the tolerance of one rounding of
    the result and of each weight.  An FP16 weight is held to 2^-25 where the largest is 2^7 or more: off by 2^-32 of
    the largest."""
    k = torch.zeros((n, width), dtype=dtype, device="cuda")
    k[0, 0] = nats
    k[1:, 8:] = 1
    others = (n - 1) * math.exp(-nats)
    want = others / (1 + others)
    u = torch.finfo(dtype).eps / 2
    tol = want * (2 * u + 2.0 ** -18) + (n * 2.0 ** -32 if dtype == torch.float16 else 0)
    return k, want, math.log1p(others) + nats, tol


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,n,nats", [(1, 100003, 17.5), (160, 3000, 17.5), (160, 3000, 12.0), (160, 200, 14.0)])
def test_absorbed_small_weights_count(dtype, B, n, nats):
    """In parts that are joined, and with all of a request's keys in one unit."""
    import glm53_flash_mlx_b200 as G

    k, want, lse64, tol = small_weights(n, nats, 576, dtype)
    pages = -(-n // 64)
    cache = torch.full((pages, 64, 576), math.nan, dtype=dtype, device="cuda")
    cache.view(-1, 576)[:n] = k
    q = torch.zeros((B, 16, 576), dtype=dtype, device="cuda")
    q[..., 0] = 1
    table = torch.arange(pages, device="cuda").int().repeat(B, 1)
    lens = torch.full((B,), n, dtype=torch.int32, device="cuda")
    out, lse = G.latent_attention_absorbed(q[..., :512], q[..., 512:], cache, table, lens, scale=1.0, return_lse=True)
    G.check_latent_status()
    assert ((out[..., 8:].double() - want).abs() <= tol).all(), (float(out[0, 0, 8]), want)
    assert ((lse.double() - lse64).abs() <= 2.0 ** -18 * (1 + lse64)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("nq", [1, 130, 200])
@pytest.mark.parametrize("n,nats", [(30000, 17.5), (30000, 16.0), (3000, 12.0), (300, 14.0)])
def test_expanded_small_weights_count(dtype, n, nats, nq):
    import glm53_flash_mlx_b200 as G

    k, want, lse64, tol = small_weights(n, nats, 128, dtype)
    q = torch.zeros((nq, 2, 128), dtype=dtype, device="cuda")
    q[..., 0] = 1
    v = k[:, None].expand(n, 2, 128)
    starts = [torch.tensor([0, m], dtype=torch.int32, device="cuda") for m in (nq, n)]
    out, lse = G.latent_attention_expanded(q, None, v, None, v, *starts, scale=1.0, causal=False, return_lse=True)
    G.check_latent_status()
    assert ((out[..., 8:].double() - want).abs() <= tol).all(), (float(out[0, 0, 8]), want)
    assert ((lse.double() - lse64).abs() <= 2.0 ** -18 * (1 + lse64)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("power", [20, 23, 24, 25, 26])
def test_weights_of_large_scores_stay_in_range(dtype, power):
    """Scores near 2^power in powers of two, where FP32 has steps of up to 8, later ones some steps above the first: no
    weight leaves its type's range.  All values are 1, and so is their mean whatever the weights: the sum of n weights
    rounded by u each, over their sum, rounded."""
    import glm53_flash_mlx_b200 as G

    u = torch.finfo(dtype).eps / 2
    i32 = dict(dtype=torch.int32, device="cuda")
    n, rises = 256, list(range(0, 41))
    k = torch.zeros((len(rises), n, 576), dtype=dtype, device="cuda")
    k[..., 0] = 2.0 ** (power - power // 2)
    k[..., 8:] = 1
    for i, x in enumerate(rises):
        k[i, 128:, 1] = x  # the second 128 keys of each request
    q = torch.zeros((len(rises), 16, 576), dtype=dtype, device="cuda")
    q[..., 0], q[..., 1] = 2.0 ** (power // 2), 1
    table = torch.arange(4 * len(rises), **i32).view(-1, 4)
    lens = torch.full((len(rises),), n, **i32)
    out = G.latent_attention_absorbed(q[..., :512], q[..., 512:], k.view(-1, 64, 576), table, lens, scale=math.log(2))
    assert ((out[..., 8:].double() - 1).abs() <= 2 * u + 2.0 ** -18).all()
    starts = torch.arange(len(rises) + 1, **i32)
    flat = k.view(-1, 1, 576)
    out = G.latent_attention_expanded(q[:, :1, :128], None, flat[..., :128], None, flat[..., 64:192], starts, starts * n,
                                      scale=math.log(2))
    assert ((out.double() - 1).abs() <= 2 * u + 2.0 ** -18).all()
    G.check_latent_status()


# --- rows without weight, rows that are not finite -------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("n", [5, 5000])  # one unit, parts that are joined
def test_absorbed_scores_of_minus_infinity(n):
    """A key whose score is -inf has no weight; a token whose keys all have such scores gives 0 and -inf, as one
    that sees no key."""
    import glm53_flash_mlx_b200 as G

    for lost in (n, n - 1, 3):  # the first `lost` keys
        ql, qr, cache, table, lens, _, rows = make_absorbed([n], [1], 16, 512, 64, 16, torch.bfloat16, n)
        qr[..., 7] = 0.5
        at = torch.arange(n, device="cuda")
        rows[0][:lost, 512 + 7] = -math.inf
        cache.view(-1, 576)[table[0].long()[at // 16] * 16 + at % 16] = rows[0]
        out, lse = G.latent_attention_absorbed(ql, qr, cache, table, lens, scale=0.05, return_lse=True)
        G.check_latent_status()
        if lost == n:
            assert (out == 0).all() and (lse == -math.inf).all()
        else:
            check(out, lse, *absorbed64(ql, qr, [rows[0][lost:]], [n - lost], [1], 0.05, torch.bfloat16))


@pytest.mark.gpu
@pytest.mark.parametrize("nq,n", [(3, 5), (200, 300), (150, 4500)])
def test_expanded_scores_of_minus_infinity(nq, n):
    import glm53_flash_mlx_b200 as G

    for lost in (n, 2, n - nq + 1):  # with the last, the first query sees keys without weight alone
        qn, qr, kn, kr, v, qs, ks = make_expanded([nq], [n], 2, 128, 64, 128, torch.bfloat16, n)
        qr, kr = qr.clone(), kr.clone()
        qr[..., 7] = 0.5
        kr[:lost, 7] = -math.inf
        out, lse = G.latent_attention_expanded(qn, qr, kn, kr, v, qs, ks, scale=0.05, return_lse=True)
        G.check_latent_status()
        none = torch.arange(nq, device="cuda") + (n - nq) + 1 <= lost
        assert (out[none] == 0).all() and (lse[none] == -math.inf).all()
        if lost < n:
            check(out, lse, *expanded64(qn, qr, kn[lost:], kr[lost:], v[lost:], [nq], [n - lost], 0.05, True, torch.bfloat16))


@pytest.mark.gpu
@pytest.mark.parametrize("what", [math.nan, math.inf])
def test_absorbed_seen_rows_that_are_not_finite(what):
    """Only the tokens that see such a row get it, through its score (NaN) or its value."""
    import glm53_flash_mlx_b200 as G

    lens, queries, H = [3000, 700, 40], [1, 3, 1], 16
    ql, qr, cache, table, n, starts, rows = make_absorbed(lens, queries, H, 512, 64, 16, torch.bfloat16, 21)
    ql.fill_(0.25)
    call = lambda: G.latent_attention_absorbed(ql, qr, cache, table, n, scale=0.05, query_starts=starts, return_lse=True)
    clean, lse = call()
    at = 698  # of the second request: its tokens see 698, 699 and 700 rows
    cache.view(-1, 576)[int(table[1, at // 16]) * 16 + at % 16, 77] = what
    got, again = call()
    G.check_latent_status()
    seen = torch.tensor([False, False, True, True, False], device="cuda")
    # an infinite score takes all weight, and inf - inf in the exponent is NaN, in 64 bits as here
    assert got[seen].isnan().all() and again[seen].isnan().all()
    assert torch.equal(got[~seen], clean[~seen]) and torch.equal(again[~seen], lse[~seen])


# --- how far results may be off on average, and counted keys ----------------


def check_average(got, lse, q, k, v, visible, scale, dtype):
    """One head's rows by their mean error.  q [n, d], k [m, d], v [m, dv], visible [n] keys each.

    Each weight's rounding is at most u of it and independent of the others, so the mean square over a row's values is
    at most u^2 sum p^2 v^2, and u^2 o^2 for the result's own (uniform errors make a third of that, which leaves room
    for the mean over as few as 64 values).  Scores: a product of d values is added up in steps of 16, each cut off at
    2^-23 of what has been added so far, below 4 standard deviations of the sum, sigma = scale sqrt(sum (q k)^2):
    e = d / 16 2^-23 4 sigma, independent from key to key.  FP16: weights are held to 2^-32 of the largest, results to
    2^-25.  Log-sums: at most the largest e, 2^-18 as above and one FP32 rounding of each of two factors."""
    u = torch.finfo(dtype).eps / 2
    q, k, v, got = q.double(), k.double(), v.double(), got.double()
    seen = torch.arange(k.shape[0], device=q.device)[None, :] < visible[:, None]
    s = torch.where(seen, (q @ k.T) * scale, -math.inf)
    log = torch.logsumexp(s, -1)
    p = torch.exp(s - log[:, None])
    out = p @ v
    e = torch.where(seen, (q.square() @ k.square().T).sqrt() * abs(scale), 0).amax(-1) * (q.shape[1] / 16 * 4 * 2.0 ** -23)
    square = (u * u + e[:, None] ** 2) * (p.square() @ v.square()) + (u * u + 2.0 ** -36) * out.square() + 1e-30
    if dtype == torch.float16:
        square = square + 2.0 ** -64 * p.amax(-1, keepdim=True) ** 2 * (seen.double() @ v.square()) + 2.0 ** -50
    err = (got - out).square().mean(-1).sqrt()
    tol = square.mean(-1).sqrt()
    bad = ~(err <= tol)
    assert not bad.any(), f"{int(bad.sum())} rows off, worst {float((err / tol).nan_to_num(nan=1e9).max()):.3f} x tolerance"
    assert ((lse.double() - log).abs() <= e + 2.0 ** -18 + 2.0 ** -22 * log.abs()).all(), float((lse - log).abs().max())


def rounded_weights(q, k, v, visible, scale, dtype, bits, drop=None):
    """Attention in 64 bits whose weights are rounded to `bits` of mantissa, rounded once to `dtype`; key `drop` left out."""
    s = (q.double() @ k.double().T) * scale
    s = s.masked_fill(torch.arange(k.shape[0])[None, :] >= visible[:, None], -math.inf)
    if drop is not None:
        s[:, drop] = -math.inf
    p = torch.exp(s - s.amax(-1, keepdim=True))
    m, x = torch.frexp(p)
    r = torch.ldexp(torch.round(m * 2.0 ** bits) / 2.0 ** bits, x)
    return ((r @ v.double()) / p.sum(-1, keepdim=True)).to(dtype), torch.logsumexp(s, -1).float()


@pytest.mark.parametrize("dtype,bits", [(torch.bfloat16, 8), (torch.float16, 11)])
@pytest.mark.parametrize("n", [1, 7, 777, 9000])
def test_mean_errors_tell_coarser_weights(dtype, bits, n):
    g = torch.Generator().manual_seed(n)
    q, k = (torch.randn((x, 576), generator=g).to(dtype) for x in (6, n))
    v, visible, scale = k[:, :512], torch.full((6,), n), 1.5 / 24
    check_average(*rounded_weights(q, k, v, visible, scale, dtype, bits), q, k, v, visible, scale, dtype)
    if n == 1:
        return
    with pytest.raises(AssertionError):  # three bits less, as of FP16 weights that are held as BF16
        check_average(*rounded_weights(q, k, v, visible, scale, dtype, bits - 3), q, k, v, visible, scale, dtype)
    with pytest.raises(AssertionError):
        check_average(*rounded_weights(q, k, v, visible, scale, dtype, bits, drop=n // 2), q, k, v, visible, scale, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,queries,H,latent,rope,page", [
    ([777], [1], 64, 512, 64, 64), ([9000], [1], 64, 512, 64, 64), ([40, 1, 3000, 500], [2, 1, 3, 1], 16, 512, 64, 16),
    ([900] * 200, [1] * 200, 16, 512, 64, 64), ([1500, 70], [1, 1], 130, 128, 0, 32)])
def test_absorbed_errors_on_average(dtype, lens, queries, H, latent, rope, page):
    import glm53_flash_mlx_b200 as G

    ql, qr, cache, table, n, starts, rows = make_absorbed(lens, queries, H, latent, rope, page, dtype, 31)
    scale = (latent + rope) ** -0.5 * 1.5
    out, lse = G.latent_attention_absorbed(ql, qr, cache, table, n, scale=scale, query_starts=starts, return_lse=True)
    G.check_latent_status()
    t = 0
    for m, nq, x in zip(lens, queries, rows):
        for j in range(nq):
            q = ql[t] if qr is None else torch.cat([ql[t], qr[t]], -1)
            vis = torch.full((H,), m - (nq - 1 - j), device="cuda")
            check_average(out[t], lse[t], q, x, x[:, :latent], vis, scale, dtype)
            t += 1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("nq,nk,H,dn,dr,dv,causal", [
    ([256], [256], 8, 192, 64, 256, True), ([129, 1, 127], [129, 640, 300], 2, 128, 64, 128, True),
    ([513], [4500], 2, 192, 64, 256, True), ([100], [3000], 2, 192, 64, 256, False), ([70] * 40, [90] * 40, 3, 64, 0, 64, True)])
def test_expanded_errors_on_average(dtype, nq, nk, H, dn, dr, dv, causal):
    import glm53_flash_mlx_b200 as G

    t = make_expanded(nq, nk, H, dn, dr, dv, dtype, 32)
    scale = (dn + dr) ** -0.5 * 1.5
    out, lse = G.latent_attention_expanded(*t, scale=scale, causal=causal, return_lse=True)
    G.check_latent_status()
    qn, qr, kn, kr, v = t[:5]
    a = b = 0
    for n, m in zip(nq, nk):
        vis = torch.arange(n, device="cuda") + (m - n) + 1 if causal else torch.full((n,), m, device="cuda")
        for h in range(H):
            q, k = qn[a:a + n, h], kn[b:b + m, h]
            if dr:
                q, k = torch.cat([q, qr[a:a + n, h]], -1), torch.cat([k, kr[b:b + m]], -1)
            check_average(out[a:a + n, h], lse[a:a + n, h], q, k, v[b:b + m, h], vis, scale, dtype)
        a, b = a + n, b + m


def check_counts(out, lse, visible):
    """Queries of 0 give every key the weight 1, so with values that mark key j in place j mod dv each value is the
    number of a place's keys over the number of all, both exact, in three roundings; a key lost or taken twice changes
    its place by one in a few dozen and the log of the number of all by more than FP32's steps there."""
    dv = out.shape[-1]
    u = torch.finfo(out.dtype).eps / 2
    vis = visible.double()[:, None]
    counts = torch.div(visible[:, None] - torch.arange(dv, device=out.device) + dv - 1, dv, rounding_mode="floor").clamp(min=0)
    want = (counts / vis.clamp(min=1))[:, None]
    assert ((out.double() - want).abs() <= (u + 2.0 ** -22) * want).all()
    some = visible > 0
    assert (lse[~some] == -math.inf).all()
    assert ((lse[some].double() - vis[some].log()).abs() <= 2.0 ** -20 + 2.0 ** -22 * vis[some].log()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,queries,H,page", [
    ([30011], [1], 16, 64), ([100003], [1], 64, 64), ([1, 63, 64, 65, 30011, 4097, 0, 777], [1] * 8, 64, 64),
    ([1, 63, 64, 65, 9011, 4097, 0, 777], [3, 2, 1, 4, 3, 3, 2, 1], 16, 16), ([5000 - 31 * i for i in range(150)], [1] * 150, 70, 8)])
def test_absorbed_counts_every_key_once(dtype, lens, queries, H, page):
    import glm53_flash_mlx_b200 as G

    ql, qr, cache, table, n, starts, _ = make_absorbed([min(x, 1) for x in lens], queries, H, 512, 64, page, dtype, 33)
    width = -(-max(lens) // page)
    # all requests read the same rows, in pages out of order
    cache = torch.full((width + 3, page, 576), math.nan, dtype=dtype, device="cuda")
    ids = torch.randperm(width + 3, device="cuda")[:width]
    at = torch.arange(max(lens), device="cuda")
    rows = torch.zeros((max(lens), 576), dtype=dtype, device="cuda")
    rows[at, at % 512] = 1
    cache.view(-1, 576)[ids[at // page] * page + at % page] = rows
    table = ids.int().repeat(len(lens), 1)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out, lse = G.latent_attention_absorbed(torch.zeros_like(ql), torch.zeros_like(qr), cache, table, n, scale=1.0,
                                           query_starts=starts, return_lse=True)
    G.check_latent_status()
    visible = [max(0, m - (nq - 1 - j)) for m, nq in zip(lens, queries) for j in range(nq)]
    check_counts(out, lse, torch.tensor(visible, device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("nq,nk,H,dv", [
    ([300, 1, 129, 0, 5], [300, 9000, 2500, 7, 2], 3, 256), ([513], [9001], 2, 128), ([1], [20003], 2, 256),
    ([128, 100], [2561, 7000], 2, 256), ([40, 130] * 80, [60, 140] * 80, 2, 64), ([300, 200], [299, 150], 2, 192)])
def test_expanded_counts_every_key_once(dtype, causal, nq, nk, H, dv):
    import glm53_flash_mlx_b200 as G

    qn, qr, kn, kr, v, qs, ks = make_expanded(nq, nk, H, 128 if dv < 256 else 192, 64, dv, dtype, 34)
    v = torch.zeros_like(v)
    at = torch.cat([torch.arange(m, device="cuda") for m in nk])
    v[torch.arange(sum(nk), device="cuda"), :, at % dv] = 1
    out, lse = G.latent_attention_expanded(torch.zeros_like(qn), torch.zeros_like(qr), kn, kr, v, qs, ks, scale=1.0,
                                           causal=causal, return_lse=True)
    G.check_latent_status()
    visible = [max(0, m - n + 1 + j) if causal else m for n, m in zip(nq, nk) for j in range(n)]
    check_counts(out, lse, torch.tensor(visible, device="cuda"))


# --- streams, graphs, together ---------------------------------------------


@pytest.mark.gpu
def test_two_graphs_and_a_side_stream():
    """Two captured decodes and an eager one on another stream share nothing: each replay gives its own
    result, with lengths that changed after the capture."""
    import glm53_flash_mlx_b200 as G

    cases = [make_absorbed([900, 40], [1, 1], 64, 512, 64, 64, torch.bfloat16, s) for s in (1, 2)]
    G.latent_attention_absorbed(*cases[0][:5], scale=0.05)
    graphs, outs = [], []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(G.latent_attention_absorbed(*c[:5], scale=0.05))
        graphs.append(g)
    for c in cases:
        c[4].copy_(torch.tensor([333, 12], dtype=torch.int32))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for g in graphs:
            g.replay()
        with torch.cuda.stream(side):
            third = G.latent_attention_absorbed(*cases[0][:5], scale=0.05)
    torch.cuda.synchronize()
    for c, o in zip(cases, outs):
        check(o, None, *absorbed64(c[0], c[1], [x[:n] for x, n in zip(c[6], (333, 12))], [333, 12], [1, 1], 0.05,
                                   torch.bfloat16))
    assert torch.equal(third, outs[0])


@pytest.mark.gpu
def test_calls_at_once_on_several_streams():
    """Both attention forms, a store and a plan, eager and as replayed graphs, on streams of their own at the
    same time: every result is the one that the call gives alone."""
    import glm53_flash_mlx_b200 as G

    dev = "cuda"
    a = make_absorbed([3000, 900, 5, 0], [1, 2, 1, 1], 64, 512, 64, 64, torch.bfloat16, 1)
    b = make_absorbed([700] * 9, [1] * 9, 16, 512, 64, 16, torch.float16, 2)
    e = make_expanded([300, 150], [300, 700], 8, 192, 64, 256, torch.bfloat16, 3)
    f = make_expanded([520], [4200], 4, 192, 64, 256, torch.bfloat16, 4)  # CTA pairs
    kv = torch.randn((40, 576), device=dev).bfloat16()
    slots = torch.randperm(64, device=dev)[:40]
    cached, new, table, free = make_plan_case(50, 16, 60, 8)

    def store():
        cache = torch.zeros((4, 16, 576), dtype=torch.bfloat16, device=dev)
        G.latent_cache_write(kv, cache, slots)
        return cache

    def plan():
        return run_plan(cached, new, table, free, len(free), 16, sum(new))[0].slots

    calls = [lambda: G.latent_attention_absorbed(*a[:5], scale=0.06, query_starts=a[5]),
             lambda: G.latent_attention_absorbed(*b[:5], scale=0.06),
             lambda: G.latent_attention_expanded(*e, scale=0.06),
             lambda: G.latent_attention_expanded(*f, scale=0.06), store, plan]
    alone = [c() for c in calls]
    torch.cuda.synchronize()
    graphs = []
    for c in calls[:5]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = c()
        graphs.append((g, out))
    streams = [torch.cuda.Stream() for _ in range(len(calls) + len(graphs))]
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        for s, c in zip(streams, calls):
            with torch.cuda.stream(s):
                got.append(c())
        for s, (g, _) in zip(streams[len(calls):], graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    G.check_latent_status()
    for i, x in enumerate(got):
        assert torch.equal(x, alone[i % len(calls)]), i
    for (_, out), want in zip(graphs, alone):
        assert torch.equal(out, want)


@pytest.mark.gpu
def test_batches_of_nothing():
    """No requests, no tokens, no keys, no pages: every row counts as one outside every request or that sees nothing."""
    import glm53_flash_mlx_b200 as G

    dev, dt = "cuda", torch.bfloat16
    i32 = dict(dtype=torch.int32, device=dev)
    new = lambda *shape: torch.full(shape, 2.0, dtype=dt, device=dev)
    none, start = torch.zeros(0, **i32), torch.zeros(1, **i32)
    for T in (0, 5):
        stale(5, 3)
        out, lse = G.latent_attention_absorbed(new(T, 3, 512), new(T, 3, 64), new(2, 16, 576), torch.zeros((0, 4), **i32),
                                               none, scale=1.0, query_starts=start, return_lse=True)
        assert out.shape == (T, 3, 512) and (out == 0).all() and (lse == -math.inf).all()
        for dv in (64, 128):
            for keys in (0, 7):
                stale(5, 3)
                out, lse = G.latent_attention_expanded(new(T, 3, 128), new(T, 3, 64), new(keys, 3, 128), new(keys, 64),
                                                       new(keys, 3, dv), start, start, scale=1.0, return_lse=True)
                assert out.shape == (T, 3, dv) and (out == 0).all() and (lse == -math.inf).all()
    # requests that hold nothing: a table without pages, a cache without pages, requests without keys
    zeros, starts = torch.zeros(5, **i32), torch.arange(6, **i32)
    for cache, table in ((new(2, 16, 576), torch.zeros((5, 0), **i32)), (new(0, 16, 576), torch.zeros((5, 2), **i32))):
        out, lse = G.latent_attention_absorbed(new(5, 3, 512), new(5, 3, 64), cache, table, zeros, scale=1.0, return_lse=True)
        assert (out == 0).all() and (lse == -math.inf).all()
    for causal in (True, False):
        out, lse = G.latent_attention_expanded(new(5, 3, 128), new(5, 3, 64), new(0, 3, 128), new(0, 64), new(0, 3, 128),
                                               starts, zeros.new_zeros(6), scale=1.0, causal=causal, return_lse=True)
        assert (out == 0).all() and (lse == -math.inf).all()
    G.check_latent_status()
    q = G.latent_cache_write(new(0, 576), new(2, 16, 576), none.long(), positions=none, queries=new(0, 3, 64),
                             inv_freq=torch.ones(32, dtype=torch.float64, device=dev))
    assert q.shape == (0, 3, 64)
    plan = G.plan_pages(none, none, torch.zeros((0, 4), **i32), none, start, page_size=16, tokens=0)
    assert plan.slots.numel() == 0 and plan.query_starts.tolist() == [0] and plan.free_count.tolist() == [0]
    G.check_latent_status()


ONE_CALL_THEN_CAPTURE = """
import torch
import glm53_flash_mlx_b200 as G

i32 = dict(dtype=torch.int32, device="cuda")
one = torch.ones(2, **i32)
table = torch.full((2, 4), -1, **i32)
plan = lambda: G.plan_pages(one * 0, one, table, torch.arange(8, **i32), one[:1] * 8, page_size=16, tokens=3)
plan()  # the one call on this device before captures
results = []
for dt in (torch.bfloat16, torch.float16):
    new = lambda *shape: torch.ones(shape, dtype=dt, device="cuda")
    for H in (16, 32, 64):
        q, cache, t = new(2, H, 576), new(4, 16, 576), torch.zeros((2, 1), **i32)
        n, e, k = one * 16, new(2, H, 256), new(32, H, 256)
        starts = torch.arange(3, **i32)
        kv, slots, pos, freq = new(2, 576), starts[:2].long(), one, torch.ones(32, dtype=torch.float64, device="cuda")
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            a = G.latent_attention_absorbed(q[..., :512], q[..., 512:], cache, t, n, scale=0.05)
            b = G.latent_attention_expanded(e, None, k, None, k, starts, starts * 16, scale=0.05)
            c = G.latent_cache_write(kv, cache, slots, positions=pos, inv_freq=freq, queries=q[..., 512:])
        g.replay()
        results.append((a, b, c))
torch.cuda.synchronize()
G.check_latent_status()
assert all((a == 1).all() and (b == 1).all() for a, b, _ in results)
print("captured")
"""


@pytest.mark.gpu
def test_capture_after_one_call_of_another_operator():
    import os
    import subprocess
    import sys
    from pathlib import Path

    root = Path(__file__).resolve().parents[1]
    env = dict(os.environ, PYTHONPATH=str(root))
    got = subprocess.run([sys.executable, "-c", ONE_CALL_THEN_CAPTURE], env=env, cwd=root, capture_output=True, text=True,
                         timeout=300)
    assert got.returncode == 0 and "captured" in got.stdout, got.stderr[-2000:]


@pytest.mark.gpu
def test_status_word_is_clear_before_any_stream_sets_it(monkeypatch):
    """The first call on a device makes the status word on its own stream; a call on another stream may run first."""
    import glm53_flash_mlx_b200 as G
    from glm53_flash_mlx_b200 import latent_attention as L

    ql, qr, cache, table, n, _, _ = make_absorbed([100, 30], [1, 1], 16, 512, 64, 16, torch.bfloat16, 9)
    bad = table.clone()
    bad[1, 1] = cache.shape[0]
    G.latent_attention_absorbed(ql, qr, cache, table, n, scale=0.05)
    monkeypatch.setattr(L, "_STATUS", {})
    first, second = torch.cuda.Stream(), torch.cuda.Stream()
    for s in (first, second):
        with torch.cuda.stream(s):  # blocks of the word's size that hold other bits, for the allocator
            blocks = [torch.full((64,), -1, dtype=torch.int32, device="cuda") for _ in range(2000)]
            del blocks
    pinned = [torch.zeros(4, dtype=torch.int32).pin_memory() for _ in range(4)]
    del pinned  # a pinned block at hand: to get a new one would wait for the device
    torch.cuda.synchronize()
    with torch.cuda.stream(first):
        torch.cuda._sleep(200_000_000)
        G.latent_attention_absorbed(ql, qr, cache, table, n, scale=0.05)
    with torch.cuda.stream(second):
        G.latent_attention_absorbed(ql, qr, cache, bad, n, scale=0.05)
    with pytest.raises(IndexError, match="page"):
        G.check_latent_status()
    G.check_latent_status()


@pytest.mark.gpu
def test_an_error_before_a_capture_is_raised_in_it():
    import glm53_flash_mlx_b200 as G

    ql, qr, cache, table, n, _, _ = make_absorbed([100, 30], [1, 1], 16, 512, 64, 16, torch.bfloat16, 9)
    call = lambda t: G.latent_attention_absorbed(ql, qr, cache, t, n, scale=0.05)
    want = call(table)
    bad = table.clone()
    bad[1, 1] = cache.shape[0]
    call(bad)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with pytest.raises(IndexError, match="page"):
        with torch.cuda.graph(g):
            call(table)
    with pytest.raises(IndexError, match="page"):  # a capture cannot clear the word
        G.check_latent_status()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call(table)
    g.replay()
    G.check_latent_status()
    assert torch.equal(out, want)


@pytest.mark.gpu
def test_views_that_are_copied_first():
    """Rows that 16-byte pieces cannot read, and integer tensors that are not contiguous, give what copies give."""
    import glm53_flash_mlx_b200 as G

    def views(x):
        wide = torch.full((*x.shape[:-1], x.shape[-1] + 9), math.nan, dtype=x.dtype, device="cuda")
        wide[..., 1:1 + x.shape[-1]] = x
        spread = torch.full((*x.shape[:-1], 2 * x.shape[-1]), math.nan, dtype=x.dtype, device="cuda")
        spread[..., ::2] = x
        turned = x.transpose(0, -1).contiguous().transpose(0, -1)
        yield from (wide[..., 1:1 + x.shape[-1]], spread[..., ::2], turned)

    def gaps(x):
        return torch.stack([x, x - 5], -1)[..., 0]

    ql, qr, cache, table, n, starts, _ = make_absorbed([100, 30, 7], [2, 1, 1], 16, 512, 64, 16, torch.bfloat16, 9)
    want = G.latent_attention_absorbed(ql, qr, cache, table, n, scale=0.05, query_starts=starts)
    for a, b in zip(views(ql), views(qr)):
        assert torch.equal(G.latent_attention_absorbed(a, b, cache, gaps(table), gaps(n), scale=0.05,
                                                       query_starts=gaps(starts)), want)
    t = make_expanded([140, 3], [200, 30], 2, 128, 64, 128, torch.bfloat16, 8)
    want = G.latent_attention_expanded(*t, scale=0.07)
    for x in zip(*(views(y) for y in t[:5])):
        assert torch.equal(G.latent_attention_expanded(*x, gaps(t[5]), gaps(t[6]), scale=0.07), want)

    kv, q = torch.randn((9, 576), device="cuda").bfloat16(), torch.randn((9, 3, 64), device="cuda").bfloat16()
    w, freq = torch.rand(512, device="cuda").bfloat16(), torch.rand(32, device="cuda", dtype=torch.float64)
    pos, slots = torch.arange(9, device="cuda").int() * 77, torch.randperm(32, device="cuda")[:9]
    store = lambda kv, q, w, pos, slots, freq: (c := torch.zeros((2, 16, 576), dtype=torch.bfloat16, device="cuda"),
                                                G.latent_cache_write(kv, c, slots, norm_weight=w, positions=pos,
                                                                     inv_freq=freq, queries=q))
    want = store(kv, q, w, pos, slots, freq)
    for a, b, c in zip(views(kv), views(q), views(w)):
        got = store(a, b, c, gaps(pos), gaps(slots), gaps(freq))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    G.check_latent_status()


@pytest.mark.gpu
def test_a_cache_past_32_bits():
    """Rows stored and read beyond 2^31 values and 2^32 bytes of the cache."""
    import glm53_flash_mlx_b200 as G

    dt, page, pages = torch.bfloat16, 64, 70000  # 2.6 x 10^9 values, 5.2 x 10^9 bytes
    cache = torch.full((pages, page, 576), math.nan, dtype=dt, device="cuda")
    lens = [300, 70]
    g = torch.Generator(device="cuda").manual_seed(3)
    ids = torch.tensor([[pages - 1, 3, 58300, pages - 2, 30000], [58255, 65000, -1, -1, -1]], dtype=torch.int32, device="cuda")
    rows = [torch.randn((m, 576), generator=g, device="cuda").to(dt) for m in lens]
    slots = torch.cat([ids[i].long()[torch.arange(m, device="cuda") // page] * page + torch.arange(m, device="cuda") % page
                       for i, m in enumerate(lens)])
    G.latent_cache_write(torch.cat(rows), cache, slots)
    assert torch.equal(cache.view(-1, 576)[slots], torch.cat(rows))
    q = torch.randn((2, 64, 576), generator=g, device="cuda").to(dt)
    out, lse = G.latent_attention_absorbed(q[..., :512], q[..., 512:], cache, ids,
                                           torch.tensor(lens, dtype=torch.int32, device="cuda"), scale=0.06, return_lse=True)
    G.check_latent_status()
    check(out, lse, *absorbed64(q[..., :512], q[..., 512:], rows, lens, [1, 1], 0.06, dt))


@pytest.mark.gpu
def test_a_prompt_batch_past_32_bits():
    """Queries, keys, values and results of more than 2^31 values each; the last requests' results against 64 bits."""
    import glm53_flash_mlx_b200 as G

    dt, H, dn, dv, B, n = torch.bfloat16, 64, 192, 256, 1100, 128  # 140,800 rows
    T = B * n
    q = torch.zeros((T, H, dn + r), dtype=dt, device="cuda")
    kv = torch.full((T, H, dn + dv), math.nan, dtype=dt, device="cuda")
    kr = torch.zeros((T, 64), dtype=dt, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(4)
    last = slice(T - 2 * n, T)
    for x in (q, kv, kr):
        x[last] = torch.randn(x[last].shape, generator=g, device="cuda").to(dt)
    kv[T - n + 70, 5, dn + 17] = math.inf  # a value that its epilogue adds again
    starts = torch.arange(B + 1, dtype=torch.int32, device="cuda") * n
    out, lse = G.latent_attention_expanded(q[..., :dn], q[..., dn:], kv[..., :dn], kr, kv[..., dn:], starts, starts,
                                           scale=0.06, return_lse=True)
    G.check_latent_status()
    got, hit = out[last].clone(), torch.zeros((2 * n, H, dv), dtype=torch.bool, device="cuda")
    hit[n + 70:, 5, 17] = True
    assert (got[hit] == math.inf).all() and out[: T - 2 * n].isnan().all()
    want = expanded64(q[last][..., :dn], q[last][..., dn:], kv[last][..., :dn], kr[last], kv[last][..., dn:], [n, n], [n, n],
                      0.06, True, dt)
    got[hit] = want[0][hit].to(dt)  # (the 64-bit form leaves out values that are not finite)
    check(got, lse[last], *want)


@pytest.mark.gpu
def test_a_second_chunk_over_the_rows_in_the_cache():
    """A prompt's next chunk attends over what is in the cache already: the keys' slots follow from the block table and
    the lengths, and the expanded form over those rows gives each query what one call over the whole prompt gives."""
    import glm53_flash_mlx_b200 as G
    from glm53_flash_mlx_b200 import synthetic as S

    dev, dt = torch.device("cuda", torch.cuda.current_device()), torch.bfloat16
    g = torch.Generator(device=dev).manual_seed(41)
    H, dn, dv, page, B = 4, 192, 256, 16, 3
    first, second = [150, 1, 64], [37, 130, 1]
    i32 = dict(dtype=torch.int32, device=dev)
    table, count = torch.full((B, 14), -1, **i32), torch.tensor([30], **i32)
    free = torch.randperm(30, generator=g, device=dev).int()
    cache = torch.full((30, page, 576), math.nan, dtype=dt, device=dev)
    freq = 10000.0 ** (-torch.arange(0, r, 2, device=dev, dtype=torch.float64) / r)
    kvb, kvb_s = S.random_block_fp8(H * (dn + dv), R, seed=5, device=dev)
    scale = (dn + r) ** -0.5

    kept, outs, cached = [[] for _ in range(B)], [], torch.zeros(B, **i32)
    for chunk in (first, second):
        T = sum(chunk)
        plan = G.plan_pages(cached, torch.tensor(chunk, **i32), table, free, count, page_size=page, tokens=T)
        kv = torch.randn((T, 576), generator=g, device=dev).to(dt)
        q = torch.randn((T, H, dn + r), generator=g, device=dev).to(dt)
        q_rope = G.latent_cache_write(kv, cache, plan.slots, positions=plan.positions, inv_freq=freq, queries=q[..., dn:])
        # the slots of all keys, cached and new
        lens = plan.seq_lens.long()
        keys = int(sum(first)) if chunk is first else sum(first) + sum(second)
        key_starts = torch.cat([lens.new_zeros(1), lens.cumsum(0)])
        request = torch.repeat_interleave(torch.arange(B, device=dev), lens, output_size=keys)
        position = torch.arange(keys, device=dev) - key_starts[request]
        key_slots = table[request, position // page].long() * page + position % page
        rows = cache.view(-1, 576)[key_slots]
        up = G.block_fp8_linear(rows[:, :R].contiguous(), kvb, kvb_s).view(keys, H, dn + dv)
        out = G.latent_attention_expanded(q[..., :dn], q_rope, up[..., :dn], rows[:, R:], up[..., dn:], plan.query_starts,
                                          key_starts.int(), scale=scale)
        check(out, None, *expanded64(q[..., :dn], q_rope, up[..., :dn], rows[:, R:], up[..., dn:], chunk, lens.tolist(),
                                     scale, True, dt))
        at = 0
        for i, n in enumerate(chunk):
            kept[i].append((q[at:at + n, :, :dn], q_rope[at:at + n], out[at:at + n]))
            at += n
        cached, count = plan.seq_lens, plan.free_count
    G.check_latent_status()
    qn, qr, want = (torch.cat([torch.cat([c[j] for c in k]) for k in kept]) for j in range(3))
    whole = G.latent_attention_expanded(qn, qr, up[..., :dn], rows[:, R:], up[..., dn:], key_starts.int(), key_starts.int(),
                                        scale=scale)
    # the same sums in another order of tiles: a rounding of the weights and one of the result on each side
    err = (whole.double() - want.double()).square().mean(-1).sqrt()
    size = want.double().square().mean(-1).sqrt()
    assert (err <= 2 * 2 * 2.0 ** -8 * size + 1e-6).all(), float((err / size).max())


@pytest.mark.gpu
def test_a_prompt_and_its_decode_together():
    """Plan, store, expand and attend a ragged prompt batch, then decode a token each: both forms give the
    layer's attention, and the output projection reads the result."""
    import glm53_flash_mlx_b200 as G
    from glm53_flash_mlx_b200 import synthetic as S

    dev, dt = torch.device("cuda", torch.cuda.current_device()), torch.bfloat16
    g = torch.Generator(device=dev).manual_seed(11)
    H, dn, dv, page = 4, 192, 256, 16
    prompts = [37, 5, 64]
    i32 = dict(dtype=torch.int32, device=dev)
    table = torch.full((3, 8), -1, **i32)
    free = torch.randperm(20, generator=g, device=dev).int()
    cache = torch.full((20, page, 576), math.nan, dtype=dt, device=dev)
    w = (1 + 0.1 * torch.randn(R, generator=g, device=dev)).to(dt)
    freq = 10000.0 ** (-torch.arange(0, r, 2, device=dev, dtype=torch.float64) / r)
    kvb, kvb_s = S.random_block_fp8(H * (dn + dv), R, seed=5, device=dev)
    ow, os_ = S.random_block_fp8(256, H * dv, seed=6, device=dev)
    scale = (dn + r) ** -0.5

    T = sum(prompts)
    zeros, count = torch.zeros(3, **i32), torch.tensor([20], **i32)
    plan = G.plan_pages(zeros, torch.tensor(prompts, **i32), table, free, count, page_size=page, tokens=T)
    kv = torch.randn((T, 576), generator=g, device=dev).to(dt)
    q = torch.randn((T, H, dn + r), generator=g, device=dev).to(dt)
    q_rope = G.latent_cache_write(kv, cache, plan.slots, norm_weight=w, positions=plan.positions, inv_freq=freq,
                                  queries=q[..., dn:])
    rows = cache.view(-1, 576)[plan.slots]
    up = G.block_fp8_linear(rows[:, :R].contiguous(), kvb, kvb_s).view(T, H, dn + dv)
    out = G.latent_attention_expanded(q[..., :dn], q_rope, up[..., :dn], rows[:, R:], up[..., dn:], plan.query_starts,
                                      plan.query_starts, scale=scale)
    check(out, None, *expanded64(q[..., :dn], q_rope, up[..., :dn], rows[:, R:], up[..., dn:], prompts, prompts, scale,
                                 True, dt))
    projected = G.block_fp8_linear(out.view(T, H * dv), ow, os_)
    head_major = out.transpose(0, 1).contiguous()
    assert torch.equal(projected, G.DSAOutputProjection().execute(head_major, ow, os_))

    # one more token each
    kv1 = torch.randn((3, 576), generator=g, device=dev).to(dt)
    q1 = torch.randn((3, H, dn + r), generator=g, device=dev).to(dt)
    step = G.plan_pages(plan.seq_lens, torch.ones(3, **i32), table, free, plan.free_count, page_size=page, tokens=3)
    qr1 = G.latent_cache_write(kv1, cache, step.slots, norm_weight=w, positions=step.positions, inv_freq=freq,
                               queries=q1[..., dn:])
    blocks = kvb.view(torch.float8_e4m3fn).float() * kvb_s.repeat_interleave(128, 0)[: kvb.shape[0]].repeat_interleave(
        128, 1)[:, :R]
    up_w = blocks.view(H, dn + dv, R)
    q_latent = torch.einsum("thd,hdr->thr", q1[..., :dn].float(), up_w[:, :dn]).to(dt)
    o = G.latent_attention_absorbed(q_latent, qr1, cache, table, step.seq_lens, scale=scale)
    G.check_latent_status()
    all_rows = [torch.cat([rows[a:b], cache.view(-1, 576)[step.slots[i:i + 1]]]) for i, (a, b) in
                enumerate(zip([0, 37, 42], [37, 42, 106]))]
    check(o, None, *absorbed64(q_latent, qr1, all_rows, [n + 1 for n in prompts], [1, 1, 1], scale, dt))
    # the expanded form of the same step: the two differ by the roundings of q_latent, the expanded keys
    # and values, both results and the values that the weights meet: at most eight roundings of 2^-8 each, a
    # relative error below 2^-5, so a cosine above 1 - 2^-10 / 2 > 0.999
    lens = [n + 1 for n in prompts]
    flat = torch.cat(all_rows)
    up1 = G.block_fp8_linear(flat[:, :R].contiguous(), kvb, kvb_s).view(-1, H, dn + dv)
    ks = torch.tensor([0, *np.cumsum(lens)], **i32)
    e = G.latent_attention_expanded(q1[..., :dn], qr1, up1[..., :dn], flat[:, R:], up1[..., dn:],
                                    torch.arange(4, **i32), ks, scale=scale)
    a = torch.einsum("thr,hdr->thd", o.float(), up_w[:, dn:])
    cos = torch.nn.functional.cosine_similarity(a.flatten(1).double(), e.flatten(1).double(), dim=-1)
    assert (cos > 0.999).all(), cos
