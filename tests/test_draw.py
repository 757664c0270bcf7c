"""nls_draw_batch: drawing tokens from typed logits, against the definition in
64 bits, and the projection and the draw together (nls_g4_lm_head_draw).

Tokens are equal. Tolerance of a probability: the kernel rounds each mass to a
multiple of 2^-45 of the largest (off by 2^-46 at most, up to 2^18 of them, in
a kept mass of at least 1: 2^-28) and the quotient, computed in fp64, once to
fp32 (2^-24): within 2^-24 + 2^-28 + 2^-40 relative.
"""
from __future__ import annotations

import numpy as np
import pytest

PROB_RTOL = 2.0 ** -24 + 2.0 ** -28 + 2.0 ** -40
DTYPES = ("f32", "f16", "bf16")


def _dt(name):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def row_running(x, p):
    """(running masses of what the settings keep, order of the whole row)."""
    t, top_p, min_p, k = float(p["temperature"]), float(p["top_p"]), float(p["min_p"]), int(p["top_k"])
    order = np.lexsort((np.arange(x.size), -x))          # descending, equal ones by index
    if t <= 0:
        return np.ones(1), order
    v = x[order]
    with np.errstate(over="ignore", invalid="ignore"):
        m = np.where(v == -np.inf, 0.0, np.exp(np.minimum((v - v[0]) / t, 0.0)))
    n = x.size
    if 0 < k < n:
        n = k
    if 0 < top_p < 1:
        run = np.cumsum(m[:n])
        n = int(np.searchsorted(run, top_p * run[-1], side="left")) + 1
    if min_p > 0:
        n = max(1, int(np.count_nonzero(m[:n] >= min_p)))
    return np.cumsum(m[:n]), order


def row_reference(x, p, u):
    """(token, probability) of one row by the definition; x float64."""
    run, order = row_running(x, p)
    if run.size == 1:
        return int(order[0]), 1.0
    at = int(np.searchsorted(run, u * run[-1], side="left"))
    t = float(p["temperature"])
    return int(order[at]), float(np.exp((x[order[at]] - x[order[0]]) / t) / run[-1])


def check(ids, probs, x, params, u):
    ids, probs = np.asarray(ids.cpu()) if hasattr(ids, "cpu") else ids, np.asarray(probs.cpu()) if hasattr(probs, "cpu") else probs
    x = x.float().cpu().numpy().astype(np.float64)
    for r in range(x.shape[0]):
        want, prob = row_reference(x[r], params[r], float(u[r]))
        assert int(ids[r]) == want, f"row {r} {params[r]} u={u[r]!r}: {ids[r]} not {want}"
        assert abs(float(probs[r]) - prob) <= PROB_RTOL * prob, f"row {r}: {probs[r]} not {prob}"


def settings(pkg, rng, n, V):
    """One of each kind of settings, with values of their own."""
    P = pkg.draw_params(n)
    for r in range(n):
        kind = r % 12
        t = rng.uniform(0.4, 1.6)
        P[r] = {0: (t, 1.0, 0.0, 40), 1: (t, 0.95, 0.05, 40), 2: (t, rng.uniform(0.05, 0.999), 0.0, 0),
                3: (t, 1.0, rng.uniform(0.001, 0.5), 0), 4: (t, 1.0, 0.0, 0), 5: (0.0, 0.9, 0.1, 5),
                6: (t, 0.9, 0.0, max(1, V // 3)), 7: (t, rng.uniform(0.3, 0.99), 0.01, 1 + V // 50),
                8: (t, 0.0, -1.0, -3), 9: (t, 0.999999, 0.0, V), 10: (t, 1e-9, 0.0, 0),
                11: (t, 0.5, 0.0, 1)}[kind]
    return P


@pytest.fixture(scope="module")
def eng(pkg):
    e = pkg.Engine(0, max_rows=1100, max_vocab=1 << 18)
    yield e
    e.close()


def test_reference_known_answers():
    p = np.zeros(1, [("temperature", "f8"), ("top_p", "f8"), ("min_p", "f8"), ("top_k", "i8")])[0]
    x = np.log(np.array([1.0, 4.0, 2.0, 2.0, 1.0]))      # masses over the largest: 1/4, 1, 1/2, 1/2, 1/4
    p["temperature"] = 1.0
    assert [row_reference(x, p, u)[0] for u in (0.0, 0.39, 0.41, 0.61, 0.81, 0.95)] == [1, 1, 2, 3, 0, 4]
    p["top_k"] = 2                                        # tokens 1, 2 (the first of the equal ones)
    assert [row_reference(x, p, u)[0] for u in (0.6, 0.7, 0.999)] == [1, 2, 2]
    assert row_reference(x, p, 0.0)[1] == pytest.approx(2 / 3)
    p["top_k"], p["top_p"] = 0, 0.5                       # 4/10 is short of it, 6/10 is not
    assert [row_reference(x, p, u)[0] for u in (0.6, 0.7)] == [1, 2]
    p["top_p"], p["min_p"] = 1.0, 0.4
    assert [row_reference(x, p, u)[0] for u in (0.45, 0.6, 0.99)] == [1, 2, 3]


def test_host_refusals(pkg):
    lib = pkg.load()
    assert lib.nls_draw_batch(None, None, 0, 8, 1, 8, None, None, None, None, 0, None) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("V", [1, 2, 3, 31, 257, 1000, 2000, 4097, 16385, 50257, 128256, 151936, 262144])
@pytest.mark.parametrize("dt", DTYPES)
def test_random_rows(pkg, eng, V, dt):
    import torch
    rng = np.random.default_rng(V)
    n = 24
    x = torch.from_numpy(rng.standard_normal((n, V)).astype(np.float32) * rng.choice([0.3, 1.0, 2.5, 8.0], (n, 1)).astype(np.float32))
    x = x.to(_dt(dt)).cuda()
    P, u = settings(pkg, rng, n, V), rng.random(n)
    ids, probs, _ = eng.draw_batch(x, P, u)
    check(ids, probs, x, P, u)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 2, 3, 7, 16, 40, 149, 300, 1100])
def test_batch_sizes(pkg, eng, rows):
    import torch
    rng = np.random.default_rng(rows)
    V = 5003
    x = torch.from_numpy((rng.standard_normal((rows, V)) * 2.5).astype(np.float32)).cuda()
    P, u = settings(pkg, rng, rows, V), rng.random(rows)
    ids, probs, _ = eng.draw_batch(x, P, u)
    check(ids, probs, x, P, u)
    # the same rows one by one
    for r in range(0, rows, max(1, rows // 5)):
        i1, p1, _ = eng.draw_batch(x[r], P[r:r + 1], u[r:r + 1])
        assert int(i1) == int(ids[r]) and float(p1) == float(probs[r])


@pytest.mark.gpu
@pytest.mark.parametrize("V", [700, 20000, 140000])
@pytest.mark.parametrize("dt", DTYPES)
def test_ties_masks_and_peaks(pkg, eng, V, dt):
    """Rows of equal logits, of few different ones, of both zeros, mostly or
    wholly but one masked by -inf or by the type's lowest value, with one token
    far above the rest, and with a long tail of tiny masses."""
    import torch
    low = float(torch.finfo(_dt(dt)).min)
    rng = np.random.default_rng(V + 1)
    base = []
    base.append(np.zeros(V))
    base.append(np.full(V, -3.25))
    base.append(rng.integers(0, 3, V).astype(np.float64))
    base.append(np.where(np.arange(V) % 2 == 0, 0.0, -0.0))
    a = np.full(V, -np.inf)
    a[V // 2] = 1.5
    base.append(a)
    a = np.full(V, low)
    a[[5, V - 1]] = (0.0, 0.25)
    base.append(a)
    base.append(np.full(V, low))
    base.append(np.where(rng.random(V) < 0.99, -np.inf, rng.standard_normal(V)))
    a = rng.standard_normal(V)
    a[V // 3] = 60.0
    base.append(a)
    a = np.full(V, -28.0)
    a[V - 2] = 0.0
    base.append(a)
    a = rng.standard_normal(V) * 1e-7 + 12.0
    base.append(a)
    a = np.full(V, low)
    a[0] = -low                                           # the widest span there is
    base.append(a)
    x = torch.from_numpy(np.stack(base)).to(_dt(dt)).repeat_interleave(12, 0).cuda()
    n = x.shape[0]
    P = settings(pkg, rng, n, V)
    u = rng.random(n)
    u[::5] = 0.0
    u[1::7] = 1.0 - 2.0 ** -53
    ids, probs, _ = eng.draw_batch(x, P, u)
    check(ids, probs, x, P, u)


@pytest.mark.gpu
def test_extreme_settings(pkg, eng):
    import torch
    rng = np.random.default_rng(11)
    V = 9001
    P = pkg.draw_params(14, temperature=[1e-300, 5e-324, 1e-3, 1e3, 1e300, np.inf, -np.inf, -1.0, 1, 1, 1, 1, 1, 1],
                        min_p=[0, 0, 0, 0, 0, 0, 0, 0, 1.0, 1.5, np.nan, 0, 0, 0],
                        top_p=[1, 1, 1, 1, 1, 0.5, 1, 1, 1, 1, np.nan, 5e-324, 1 - 2.0 ** -53, 2.0],
                        top_k=[0, 0, 0, 0, 0, 0, 0, 0, 0, 0, -2**63, 0, 0, 2**63 - 1])
    x = torch.from_numpy((rng.standard_normal((14, V)) * 2).astype(np.float32)).cuda()
    u = rng.random(14)
    ids, probs, _ = eng.draw_batch(x, P, u)
    check(ids, probs, x, P, u)


@pytest.mark.gpu
@pytest.mark.parametrize("k", [1, 2, 63, 255, 256, 257, 1000, 1024, 1025, 2048, 2049, 5000, 19999, 20000, 20001])
def test_top_k_borders(pkg, eng, k):
    """Every border of top-k, over equal logits too (half-precision rows)."""
    import torch
    rng = np.random.default_rng(k)
    V, n = 20000, 9
    x = torch.from_numpy((rng.standard_normal((n, V)) * 2).astype(np.float32))
    x[3:6] = x[3:6].bfloat16().float()
    x[6] = torch.round(x[6])
    x = x.cuda()
    P = pkg.draw_params(n, temperature=[0.3, 1, 3] * 3, top_k=k, top_p=[1, 0.9, 0.99, 0.9, 1, 1, 1, 0.5, 1])
    u = rng.random(n)
    u[4] = 1 - 2.0 ** -53
    ids, probs, _ = eng.draw_batch(x, P, u)
    check(ids, probs, x, P, u)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
def test_strides_alignment_and_host_rows(pkg, eng, dt):
    import torch
    rng = np.random.default_rng(3)
    wide = torch.from_numpy((rng.standard_normal((13, 30011)) * 2).astype(np.float32)).to(_dt(dt)).cuda()
    for off, V in ((0, 30011), (1, 30000), (3, 4099), (5, 11), (8, 29000), (30010, 1)):
        x = wide[:, off:off + V]
        P, u = settings(pkg, rng, 13, V), rng.random(13)
        ids, probs, _ = eng.draw_batch(x, P, u)
        check(ids, probs, x, P, u)
        hi, hp, _ = eng.draw_batch(x.cpu(), P, u)
        assert np.array_equal(hi, ids.cpu().numpy()) and np.array_equal(hp, probs.cpu().numpy())
    xs = wide[:, ::2]                                      # columns apart: copied
    P, u = settings(pkg, rng, 13, xs.shape[1]), rng.random(13)
    ids, probs, _ = eng.draw_batch(xs, P, u)
    check(ids, probs, xs, P, u)
    assert eng.draw_batch(wide[:0], pkg.draw_params(0), np.zeros(0))[0].numel() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("V", [300, 70000])
def test_bad_rows(pkg, eng, V):
    """Rows that cannot be drawn from fail alone."""
    import torch
    x = torch.zeros((8, V))
    x[1, V - 1] = float("nan")
    x[2, 0] = float("inf")
    x[3] = float("-inf")
    x[6, 10] = float("nan")
    P = pkg.draw_params(8, temperature=[1, 1, 1, 1, float("nan"), 1, 0, 0], top_k=[0, 5, 0, 0, 0, 3, 0, 0])
    u = np.array([0.5, 0.5, 0.5, 0.5, 0.5, 1.0, 0.5, float("nan")])
    ids, probs, st = eng.draw_batch(x.cuda(), P, u, check=False)
    torch.cuda.synchronize()
    assert ids.tolist() == [V // 2 - 1, -1, -1, -1, -1, -1, -1, 0]
    assert probs.tolist()[1:] == [0, 0, 0, 0, 0, 0, 1]
    with pytest.raises(pkg.NlsError) as e:
        eng.draw_batch(x[1:2].cuda(), P[1:2], u[1:2])
    assert e.value.status == pkg._abi.NLS_ERR_NAN_LOGITS
    with pytest.raises(pkg.NlsError) as e:
        eng.draw_batch(x[:1].cuda(), P[:1])                # no uniform
    assert e.value.status == pkg._abi.NLS_ERR_INVALID_ARG
    ids, probs, _ = eng.draw_batch(x[:1].cuda(), pkg.draw_params(1, temperature=0.0))
    assert ids.tolist() == [0]
    # the handle is as before
    ids, _, _ = eng.draw_batch(x[:1].cuda(), P[:1], u[:1])
    assert ids.tolist() == [V // 2 - 1]


@pytest.mark.gpu
def test_device_refusals(pkg, eng):
    import torch
    lib = pkg.load()
    x = torch.zeros((2, 64), device="cuda")
    P = torch.zeros(64, dtype=torch.uint8, device="cuda")
    u = torch.zeros(2, dtype=torch.float64, device="cuda")
    ids = torch.full((2,), 9, dtype=torch.int64, device="cuda")

    def call(xp=x.data_ptr(), lt=0, ld=64, rows=2, V=64, pp=P.data_ptr(), ip=ids.data_ptr(), flags=3):
        return lib.nls_draw_batch(eng._h, xp, lt, ld, rows, V, pp, u.data_ptr(), ip, None, flags, None)

    for bad in (dict(xp=None), dict(xp=x.data_ptr() + 1), dict(lt=3), dict(ld=63), dict(rows=-1), dict(V=0),
                dict(pp=None), dict(ip=None), dict(flags=4)):
        assert call(**bad) == 1, bad
    assert call(rows=1101) == 6 and call(V=(1 << 18) + 1, ld=1 << 19) == 6
    assert call(rows=0) == 0
    torch.cuda.synchronize()
    assert ids.tolist() == [9, 9]
    with pytest.raises(ValueError):
        eng.draw_batch(x, pkg.draw_params(3), np.zeros(2))
    with pytest.raises(ValueError):
        eng.draw_batch(x, pkg.draw_params(2), torch.zeros(2, device="cuda"))
    with pytest.raises(TypeError):
        eng.draw_batch(x.double(), pkg.draw_params(2), np.zeros(2))


@pytest.mark.gpu
def test_same_as_the_reference_sampler_away_from_borders(pkg, eng, engine):
    """nls_sample_batch's chain on the same rows: the two differ only by the
    reference's fp32 rounding of sums (and by ties at the top-k border), so on
    4096 tokens almost every draw is the same token."""
    rng = np.random.default_rng(17)
    B, V = 400, 4096
    x = (rng.standard_normal((B, V)) * 2.5).astype(np.float32)
    P = pkg.draw_params(B, temperature=rng.uniform(0.5, 1.2, B), top_k=rng.choice([0, 20, 100], B),
                        top_p=rng.uniform(0.8, 1.0, B), min_p=rng.choice([0.0, 0.05], B))
    R = np.zeros(B, pkg.ROW_PARAMS_DTYPE)
    for name in P.dtype.names:
        R[name] = P[name]
    R["repeat_penalty"] = 1.0
    u = rng.random(B)
    ids, _, _ = eng.draw_batch(x, P, u)
    ref, _, _ = engine.sample_batch(x, R, uniforms=u)
    # the reference's sums of up to 4096 fp32 terms (the softmax's, top-p's and
    # the draw's) are each off by 4096 * 2^-24 relative at most: a token of its
    # own choice lies that near to u times the kept mass
    slack = 3 * V * 2.0 ** -24
    for r in np.nonzero(ids != ref)[0]:
        run, order = row_running(x[r].astype(np.float64), P[r])
        at = int(np.nonzero(order == ref[r])[0][0])
        lo, hi = (run[at - 1] if at else 0.0), run[min(at, run.size - 1)]
        assert lo - slack * run[-1] <= u[r] * run[-1] <= hi + slack * run[-1]


@pytest.mark.gpu
def test_streams_and_graphs(pkg, eng):
    import torch
    rng = np.random.default_rng(21)
    B, V = 6, 33333
    x = torch.from_numpy((rng.standard_normal((B, V)) * 2).astype(np.float32)).bfloat16().cuda()
    P, u = settings(pkg, rng, B, V), torch.from_numpy(rng.random(B)).cuda()
    Pd = torch.from_numpy(P.view(np.uint8).copy()).cuda()
    ids = torch.zeros(B, dtype=torch.int64, device="cuda")
    probs = torch.zeros(B, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    i2, p2, _ = eng.draw_batch(x, P, u, stream=side.cuda_stream)
    check(i2, p2, x, P, u.cpu().numpy())
    graph = torch.cuda.CUDAGraph()
    eng.draw_batch(x, Pd, u, out_ids=ids, out_probs=probs)
    with torch.cuda.graph(graph):
        eng.draw_batch(x, Pd, u, out_ids=ids, out_probs=probs, check=False)
    for _ in range(3):
        x.copy_(torch.from_numpy((rng.standard_normal((B, V)) * 2).astype(np.float32)))
        u.copy_(torch.from_numpy(rng.random(B)))
        graph.replay()
        torch.cuda.synchronize()
        check(ids, probs, x, P, u.cpu().numpy())
    del graph


@pytest.mark.gpu
@pytest.mark.parametrize("nb,lt", [(1, "f32"), (5, "bf16"), (40, "f16")])
def test_projection_and_draw_together(pkg, eng, nb, lt):
    """A decode step's tail in one call equals its two calls, and its tokens
    are those of the definition on the projection's own logits."""
    import torch
    g = torch.Generator().manual_seed(nb)
    weight = torch.randn((20011, 512), generator=g) * 0.08
    w = pkg.g4_quantize(weight.cuda(), group=64, symmetric=nb != 5, dtype=torch.float16)
    x = torch.randn((nb, 512), generator=g).half().cuda()
    rng = np.random.default_rng(nb)
    P, u = settings(pkg, rng, nb, 20011), rng.random(nb)
    logits = eng.g4_matmul(w, x, out_dtype=_dt(lt))
    ids, probs, _ = eng.draw_batch(logits, P, u)
    check(ids, probs, logits, P, u)
    i2, p2, _ = eng.g4_lm_head_draw(w, x, P, u, logits_dtype=_dt(lt))
    assert torch.equal(ids, i2) and torch.equal(probs, p2)
    i3, p3, _ = eng.g4_lm_head_draw(w, x.cpu(), P, u, logits_dtype=_dt(lt))
    assert np.array_equal(i3, ids.cpu().numpy()) and np.array_equal(p3, probs.cpu().numpy())
    with pytest.raises(pkg.NlsError):
        eng.g4_lm_head_draw(w, torch.zeros((1101, 512), device="cuda"), pkg.draw_params(1101), np.zeros(1101))
    bad = x.clone()
    bad[0, 0] = float("nan")
    with pytest.raises(pkg.NlsError):
        eng.g4_lm_head_draw(w, bad, P, u)


@pytest.mark.gpu
def test_a_generation_loop(pkg, eng):
    """Steps of a small model: hidden state from the last token, projection,
    draw, all on one stream without waiting in between."""
    import torch
    g = torch.Generator().manual_seed(0)
    V, D, B, steps = 5000, 256, 3, 12
    table = torch.randn((V, D), generator=g).half().cuda()
    w = pkg.g4_quantize(torch.randn((V, D), generator=g).cuda() * 0.2, group=128, dtype=torch.float16)
    P = pkg.draw_params(B, temperature=[0.7, 1.0, 0.0], top_k=[40, 0, 0], top_p=[0.95, 0.9, 1.0])
    Pd = torch.from_numpy(P.view(np.uint8).copy()).cuda()
    rng = np.random.default_rng(1)
    us = torch.from_numpy(rng.random((steps, B))).cuda()
    tok = torch.tensor([1, 2, 3], device="cuda")
    seen = []
    for t in range(steps):
        tok, _, _ = eng.g4_lm_head_draw(w, table[tok], Pd, us[t], logits_dtype=torch.float32, check=False)
        seen.append(tok)
    tok = torch.tensor([1, 2, 3], device="cuda")
    for t in range(steps):
        logits = eng.g4_matmul(w, table[tok], out_dtype=torch.float32)
        x = logits.cpu().numpy().astype(np.float64)
        want = [row_reference(x[r], P[r], float(us[t, r]))[0] for r in range(B)]
        assert seen[t].tolist() == want
        tok = seen[t]


@pytest.mark.gpu
@pytest.mark.parametrize("nb", [2, 20])
def test_a_captured_step(pkg, eng, nb):
    """Projection and draw captured together, replayed on new inputs, also after
    a larger call on the handle."""
    import torch
    g = torch.Generator().manual_seed(nb)
    V, D = 9001, 512
    w = pkg.g4_quantize(torch.randn((V, D), generator=g).cuda() * 0.1, group=64, symmetric=False, dtype=torch.float16)
    rng = np.random.default_rng(nb)
    P = settings(pkg, rng, nb, V)
    Pd = torch.from_numpy(P.view(np.uint8).copy()).cuda()
    x, u = torch.randn((nb, D), generator=g).half().cuda(), torch.from_numpy(rng.random(nb)).cuda()
    ids = torch.zeros(nb, dtype=torch.int64, device="cuda")
    probs = torch.zeros(nb, device="cuda")
    fresh = pkg.Engine(0, max_rows=256, max_vocab=1 << 14)
    graph = torch.cuda.CUDAGraph()
    try:
        fresh.g4_lm_head_draw(w, x, Pd, u, logits_dtype=torch.float32, out_ids=ids, out_probs=probs)
        with torch.cuda.graph(graph):
            fresh.g4_lm_head_draw(w, x, Pd, u, logits_dtype=torch.float32, out_ids=ids, out_probs=probs, check=False)
        many = torch.randn((250, D), generator=g).half().cuda()
        fresh.g4_lm_head_draw(w, many, pkg.draw_params(250, top_k=5), np.full(250, 0.5), logits_dtype=torch.float32)
        for _ in range(3):
            x.copy_(torch.randn((nb, D), generator=g).half())
            u.copy_(torch.from_numpy(rng.random(nb)))
            graph.replay()
            torch.cuda.synchronize()
            logits = eng.g4_matmul(w, x, out_dtype=torch.float32)
            check(ids, probs, logits, P, u.cpu().numpy())
    finally:
        del graph
        fresh.close()


@pytest.mark.gpu
def test_two_handles_at_once(pkg, eng):
    """Calls on two handles and two streams, side by side."""
    import torch
    g = torch.Generator().manual_seed(3)
    V, D, steps = 30011, 1024, 20
    w = pkg.g4_quantize(torch.randn((V, D), generator=g).cuda() * 0.1, group=128, dtype=torch.float16)
    sizes = (3, 24)
    rng = np.random.default_rng(3)
    P = [settings(pkg, rng, n, V) for n in sizes]
    Pd = [torch.from_numpy(p.view(np.uint8).copy()).cuda() for p in P]
    x = [torch.randn((steps, n, D), generator=g).half().cuda() for n in sizes]
    u = [torch.from_numpy(rng.random((steps, n))).cuda() for n in sizes]
    want = [[eng.g4_lm_head_draw(w, x[i][t], Pd[i], u[i][t], logits_dtype=torch.bfloat16)[:2] for t in range(steps)]
            for i in range(2)]
    handles = [pkg.Engine(0, max_rows=32, max_vocab=1 << 15) for _ in sizes]
    streams = [torch.cuda.Stream() for _ in sizes]
    try:
        for i in range(2):  # (the workspaces)
            handles[i].g4_lm_head_draw(w, x[i][0], Pd[i], u[i][0], logits_dtype=torch.bfloat16)
        torch.cuda.synchronize()
        got = [[], []]
        for t in range(steps):
            for i in range(2):
                with torch.cuda.stream(streams[i]):
                    got[i].append(handles[i].g4_lm_head_draw(w, x[i][t], Pd[i], u[i][t], logits_dtype=torch.bfloat16,
                                                             check=False)[:2])
        torch.cuda.synchronize()
        for i in range(2):
            for t in range(steps):
                assert torch.equal(got[i][t][0], want[i][t][0]) and torch.equal(got[i][t][1], want[i][t][1])
    finally:
        for h in handles:
            h.close()


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["params", "uniforms", "out_ids", "out_probs"])
def test_misaligned_device_arrays_are_refused(pkg, eng, which):
    """Before anything is launched; host arrays may lie anywhere."""
    import ctypes
    import torch
    lib = pkg.load()
    w = pkg.g4_quantize(torch.ones((64, 128), device="cuda"), group=128)
    x = torch.zeros((2, 128), device="cuda")
    at = {n: torch.zeros(128, dtype=torch.uint8, device="cuda") for n in ("params", "uniforms", "out_ids", "out_probs")}
    ptr = [t.data_ptr() + (2 if n == which == "out_probs" else 4 if n == which else 0) for n, t in at.items()]
    assert lib.nls_draw_batch(eng._h, x.data_ptr(), 0, 64, 2, 64, *ptr, 3, None) == 1
    assert lib.nls_g4_lm_head_draw(eng._h, ctypes.byref(w.struct), x.data_ptr(), 0, 128, 2, 0, *ptr, 3, None) == 1
    if which == "params":
        with pytest.raises(pkg.NlsError) as e:
            eng.draw_batch(x, at["params"][4:68], torch.zeros(2, dtype=torch.float64, device="cuda"))
        assert e.value.status == pkg._abi.NLS_ERR_INVALID_ARG
    host = np.zeros(256, np.uint8)
    host[1:65] = pkg.draw_params(2).view(np.uint8)
    base = host.ctypes.data + 1
    logits = np.zeros((2, 64), np.float32)
    assert lib.nls_draw_batch(eng._h, logits.ctypes.data, 0, 64, 2, 64, base, base + 64, base + 80, base + 96, 0, None) == 0
    assert host[81:97].view(np.int64).tolist() == [0, 0]


@pytest.mark.gpu
def test_an_empty_batch_has_no_error_of_an_earlier_call(pkg, eng):
    import torch
    w = pkg.g4_quantize(torch.ones((64, 128), device="cuda"), group=128)
    x = torch.zeros((2, 128), device="cuda")
    nan = torch.full((1, 64), float("nan"), device="cuda")
    P, u = pkg.draw_params(1), np.zeros(1)
    none, no_u = pkg.draw_params(0), np.zeros(0)
    for empty in (lambda: eng.draw_batch(nan[:0], none, no_u)[0].numel(),
                  lambda: eng.g4_matmul(w, x[:0]).numel(),
                  lambda: eng.g4_lm_head_draw(w, x[:0], none, no_u)[0].numel()):
        ids, _, _ = eng.draw_batch(nan, P, u, check=False)
        assert empty() == 0
        assert ids.tolist() == [-1]
        with pytest.raises(pkg.NlsError):                  # (the earlier call's error is its own)
            eng.draw_batch(nan, P, u)


@pytest.mark.gpu
def test_profiled_times_are_the_last_draws(pkg):
    """A draw is a sampling call: with profiling on its times replace those of
    the call before, and with profiling off there are none."""
    import torch
    e = pkg.Engine(0, max_rows=512, max_vocab=1 << 17)
    try:
        w = pkg.g4_quantize(torch.ones((64, 128), device="cuda"), group=128)
        big = torch.randn((512, 100000), device="cuda")
        P, u = pkg.draw_params(512, top_p=0.9), np.full(512, 0.5)
        e.draw_batch(big, P, u)
        with pytest.raises(pkg.NlsError):
            e.last_kernel_ms()
        e.set_profiling(True)
        for _ in range(2):
            e.draw_batch(big, P, u)
            many = e.last_kernel_ms()
            # (three events, recorded one after the other behind the one kernel;
            # 205 MB cannot be read in less)
            assert 0.02 < many[0] <= many[1] <= many[2]
            e.draw_batch(big[:1, :64], P[:1], u[:1])
            one = e.last_kernel_ms()
            assert 0 < one[2] < many[2]
            e.draw_batch(big, P, u)
            e.g4_lm_head_draw(w, torch.zeros((1, 128), device="cuda"), P[:1], u[:1])
            assert 0 < e.last_kernel_ms()[2] < many[2]
        e.set_profiling(False)
        e.draw_batch(big, P, u)
        with pytest.raises(pkg.NlsError):
            e.last_kernel_ms()
    finally:
        e.close()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [2, 40, 300])
def test_probability_of_a_token_among_many_equal_ones(pkg, eng, rows):
    """More equal logits at a border than are collected: the kept mass is the one
    that the selection over the whole row finds, not an earlier estimate."""
    import torch
    V = 60000
    x = torch.zeros((rows, V), device="cuda")
    x[:, ::3] = -1.0
    x[:, 7] = 2.0
    P = pkg.draw_params(rows, temperature=1.0, top_p=0.5, min_p=[0.0, 0.2] * (rows // 2), top_k=[0, 9001] * (rows // 2))
    u = np.random.default_rng(rows).random(rows)
    ids, probs, _ = eng.draw_batch(x, P, u)
    check(ids, probs, x, P, u)


def draw_us(eng, x, P, u):
    """The least of some calls' device times, L2 flushed before each."""
    import torch
    P = torch.from_numpy(P.view(np.uint8).copy()).cuda()
    u = torch.from_numpy(u).cuda()
    flush = torch.empty(1 << 28, dtype=torch.uint8, device="cuda")
    best = float("inf")
    for _ in range(6):
        flush.zero_()
        a, b = torch.cuda.Event(True), torch.cuda.Event(True)
        a.record()
        eng.draw_batch(x, P, u, check=False)
        b.record()
        b.synchronize()
        best = min(best, a.elapsed_time(b) * 1e3)
    return best


@pytest.mark.gpu
@pytest.mark.parametrize("rows,dt", [(4, "f32"), (64, "bf16"), (256, "f32")])
@pytest.mark.parametrize("T", [0.05, 0.1, 0.2])
def test_top_k_beyond_the_tokens_with_mass(pkg, eng, rows, dt, T):
    """Low temperatures leave fewer tokens with a mass than top-k keeps: all of
    them are kept, and no row goes to the selection over the whole row."""
    import torch
    V = 128256
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = (torch.randn((rows, V), generator=g, device="cuda") * 2.5).to(_dt(dt))
    u = np.random.default_rng(rows).random(rows)
    plain = draw_us(eng, x, pkg.draw_params(rows, temperature=T, top_p=0.999), u)
    for k in (300, 400, 600, 1000, 3000, 5000, 20000):
        for top_p in (1.0, 0.9):
            P = pkg.draw_params(rows, temperature=T, top_k=k, top_p=top_p)
            ids, probs, _ = eng.draw_batch(x, P, u)
            some = [0, rows // 2, rows - 1]
            check(ids[some], probs[some], x[some], P[some], u[some])
            us = draw_us(eng, x, P, u)
            assert us < 4 * plain, f"top-k {k}: {us} us, without it {plain} us"


@pytest.mark.gpu
@pytest.mark.parametrize("rows,dt,keep", [(64, "bf16", (0, 75000)), (64, "bf16", (0, 120000)), (64, "f16", (75001, 150001)),
                                          (40, "bf16", (1, 75003)), (16, "f32", (60000, 90000)), (2, "f32", (140000, 150001))])
def test_a_row_whose_tokens_lie_in_one_part(pkg, eng, rows, dt, keep):
    """All else masked: the CTA of that part collects all there is to collect,
    and no row goes to the selection over the whole row."""
    import torch
    V = 150001
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = torch.randn((rows, V), generator=g, device="cuda").to(_dt(dt))
    y = torch.full_like(x, -float("inf"))
    y[:, keep[0]:keep[1]] = x[:, keep[0]:keep[1]]
    u = np.random.default_rng(rows).random(rows)
    for P in (pkg.draw_params(rows, top_p=0.9), pkg.draw_params(rows, top_k=1500, top_p=0.95)):
        ids, probs, _ = eng.draw_batch(y, P, u)
        some = np.unique(np.linspace(0, rows - 1, 12).astype(int))
        check(ids[some], probs[some], y[some], P[some], u[some])
        plain, us = draw_us(eng, x, P, u), draw_us(eng, y, P, u)
        assert us < 4 * plain, f"{us} us, without a mask {plain} us"


@pytest.mark.gpu
@pytest.mark.parametrize("rows,dt", [(4, "f32"), (64, "bf16"), (64, "f16"), (200, "f32")])
@pytest.mark.parametrize("std,given", [(1.0, dict(top_p=0.9)), (2.5, dict(temperature=2.0, top_p=0.95)),
                                       (1.0, dict(temperature=1.5, min_p=0.01))])
def test_masked_logits_do_not_slow_a_row_down(pkg, eng, rows, dt, std, given):
    """Logits masked by a finite value or by -inf, a few or many, anywhere in the
    row: the same tokens as the definition's, and no row goes to the selection
    over the whole row, which takes twenty times as long."""
    import torch
    V = 150001
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = (torch.randn((rows, V), generator=g, device="cuda") * std).to(_dt(dt))
    rng = np.random.default_rng(rows)
    P, u = pkg.draw_params(rows, **given), rng.random(rows)
    plain = draw_us(eng, x, P, u)
    low = float(torch.finfo(_dt(dt)).min)
    for what in (slice(0, 1), slice(77, 78), slice(0, 40000), slice(0, 140000), slice(120000, V), slice(0, V, 2)):
        for value in (low, -float("inf"), -3e4):
            y = x.clone()
            y[:, what] = value
            ids, probs, _ = eng.draw_batch(y, P, u)
            some = [0, rows // 2, rows - 1]
            check(ids[some], probs[some], y[some], P[some], u[some])
            us = draw_us(eng, y, P, u)
            assert us < 4 * plain, f"{what} {value}: {us} us, without a mask {plain} us"


@pytest.mark.gpu
@pytest.mark.parametrize("rows,V,dt", [(256, 128256, "f32"), (64, 151936, "bf16"), (8, 262144, "f16")])
@pytest.mark.parametrize("T,min_p", [(1.0, 0.02), (1.2, 0.05), (1.0, 0.1)])
def test_min_p_that_keeps_many_tokens(pkg, eng, rows, V, dt, T, min_p):
    """The border of min-p in a crowded bin: no row goes to the selection over
    the whole row."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = torch.randn((rows, V), generator=g, device="cuda").to(_dt(dt))
    rng = np.random.default_rng(rows)
    plain = draw_us(eng, x, pkg.draw_params(rows, temperature=T), rng.random(rows))
    P = pkg.draw_params(rows, temperature=T, min_p=min_p)
    for _ in range(4):
        u = rng.random(rows)
        ids, probs, _ = eng.draw_batch(x, P, u)
        some = np.unique(np.linspace(0, rows - 1, 12).astype(int))
        check(ids[some], probs[some], x[some], P[some], u[some])
        us = draw_us(eng, x, P, u)
        assert us < 4 * plain, f"{us} us, without min-p {plain} us"


@pytest.mark.gpu
@pytest.mark.parametrize("rows,dt", [(1, "f32"), (64, "bf16"), (300, "f16")])
def test_a_row_of_equal_logits_takes_a_bounded_time(pkg, eng, rows, dt):
    """The selection over the whole row: some twenty passes over it by one CTA, so
    that a hundred times as long as a row that is read twice is a wide bound; with
    the additions of equal logits one after the other it was seven hundred."""
    import torch
    V = 150001
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = (torch.randn((rows, V), generator=g, device="cuda") * 2.5).to(_dt(dt))
    y = torch.full_like(x, 0.75)
    u = np.random.default_rng(rows).random(rows)
    P = pkg.draw_params(rows, top_p=0.9, min_p=[0.0, 0.3][rows % 2], top_k=70000)
    ids, probs, _ = eng.draw_batch(y, P, u)
    some = np.unique(np.linspace(0, rows - 1, 6).astype(int))
    check(ids[some], probs[some], y[some], P[some], u[some])
    plain, us = draw_us(eng, x, P, u), draw_us(eng, y, P, u)
    assert us < 100 * plain, f"{us} us, other rows {plain} us"
