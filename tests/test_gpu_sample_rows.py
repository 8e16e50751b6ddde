"""Row sampling on the GPU against a 64-bit restatement.  Tokens and counts
are equal: weights are summed exactly as multiples of 2^-45, so a draw differs
only if u lies within n * 2^-45 of a border (1e-8 for the longest row)."""
import numpy as np
import pytest

import serving_ref as R
from conftest import has_gpu

pytestmark = pytest.mark.gpu
if has_gpu():
    import torch

    TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def run(qtts, logits, u, temperature=None, top_k=None, top_p=None, min_p=None, dtype="f32", ld=0, stream=0):
    n, V = logits.shape[0], logits.shape[1]
    t = {"u": torch.from_numpy(np.asarray(u, np.float32)).cuda()}
    for name, v, ty in (("temperature", temperature, np.float32), ("top_k", top_k, np.int32), ("top_p", top_p, np.float32),
                        ("min_p", min_p, np.float32)):
        if v is not None:
            t[name] = torch.from_numpy(np.broadcast_to(np.asarray(v, ty), (n,)).copy()).cuda()
    token, kept = (torch.full((n,), -7, dtype=torch.int32, device="cuda") for _ in range(2))
    logprob = torch.full((n,), 7.0, device="cuda")
    torch.cuda.synchronize()
    qtts.sample_rows_dev(logits.data_ptr(), n, V, t["u"].data_ptr(), token.data_ptr(), dtype=dtype,
                         kept_ptr=kept.data_ptr(), logprob_ptr=logprob.data_ptr(), ld=ld, stream=stream,
                         **{k + "_ptr": v.data_ptr() for k, v in t.items() if k != "u"})
    torch.cuda.synchronize()
    return token.cpu().numpy(), kept.cpu().numpy(), logprob.cpu().numpy()


def check(qtts, x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, dtype="f32", ld=0):
    """x: f32 numpy rows; every row against the restatement."""
    n, V = x.shape
    full = torch.zeros(n, max(ld, V), dtype=TYPES[dtype], device="cuda")
    full[:, :V] = torch.from_numpy(x).cuda().to(TYPES[dtype])
    tok, kept, lp = run(qtts, full[:, :V], u, temperature, top_k, top_p, min_p, dtype, ld)
    seen = full[:, :V].float().cpu().numpy()
    b = lambda v: np.broadcast_to(np.asarray(v, np.float32), (n,))  # noqa: E731
    T, K, P, M = b(temperature), np.broadcast_to(np.asarray(top_k), (n,)), b(top_p), b(min_p)
    for r in range(n):
        wt, wk, wl, margin = R.sample(seen[r], T[r], int(K[r]), P[r], M[r], u[r])
        assert kept[r] == wk, (r, kept[r], wk)
        if margin <= V * 2.0 ** -45:
            continue
        assert tok[r] == wt, (r, tok[r], wt, margin)
        # log of a weight that is off by half of 2^-45 and rounded to f32
        if np.isinf(wl):
            assert lp[r] == wl
        else:
            assert abs(lp[r] - wl) <= 2.0 ** -24 * abs(wl) + 2.0 ** -46 * (np.exp(min(30.0, -wl)) + V) + 1e-12, (r, lp[r], wl)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V", [1, 2, 31, 32, 33, 100, 1000, 2048, 2049, 4000, 5000, 40000])
def test_filters(qtts, V, dtype):
    rng = np.random.default_rng(V)
    n = 24
    x = (rng.standard_normal((n, V)) * 3).astype(np.float32)
    x[:, rng.integers(0, V, V // 7)] = -np.inf if V > 20 else 0.0
    check(qtts, x, rng.random(n).astype(np.float32), temperature=rng.choice([0.3, 0.8, 1.0, 1.7], n),
          top_k=rng.choice([0, 1, 2, 7, 50, V - 1, V, V + 5], n), top_p=rng.choice([0.0, 0.1, 0.5, 0.9, 0.999, 1.0], n),
          min_p=rng.choice([0.0, 0.001, 0.05, 0.5, 1.0, 3.0], n), dtype=dtype)


@pytest.mark.parametrize("V,dtype,n", [(151936, "f32", 5), (151936, "bf16", 20), (262144, "f16", 3), (70001, "f32", 9)])
@pytest.mark.parametrize("spread", [0.5, 3.0])
def test_long_rows(qtts, V, dtype, n, spread):
    rng = np.random.default_rng(V + n)
    x = (rng.standard_normal((n, V)) * spread).astype(np.float32)
    check(qtts, x, rng.random(n).astype(np.float32), temperature=rng.choice([0.7, 1.0, 1.3], n),
          top_k=rng.choice([0, 0, 50, 1000, 60000], n), top_p=rng.choice([0.3, 0.9, 0.95, 1.0], n),
          min_p=rng.choice([0.0, 0.0, 0.02], n), dtype=dtype, ld=V + 3)


@pytest.mark.parametrize("V", [40, 2048, 30000])
def test_ties_keep_the_lowest_indices(qtts, V):
    rng = np.random.default_rng(V)
    n = 16
    x = rng.integers(0, 3, (n, V)).astype(np.float32)
    x[0] = 1.5  # every token the same
    check(qtts, x, rng.random(n).astype(np.float32), temperature=0.9, top_k=rng.choice([0, 3, V // 2, V], n),
          top_p=rng.choice([0.2, 0.6, 1.0], n))
    check(qtts, x, rng.random(n).astype(np.float32), temperature=0.0)


def test_special_logits(qtts):
    V = 300
    rng = np.random.default_rng(5)
    x = rng.standard_normal((12, V)).astype(np.float32)
    x[0] = -np.inf
    x[1] = np.nan
    x[2] = -np.inf
    x[2, 17] = -3.0e38
    x[3, ::3] = np.nan
    x[4, 5] = np.inf
    x[5, [7, 9, 200]] = np.inf
    x[6] = 0.0
    x[6, ::2] = -0.0
    x[7] = -1e30
    x[7, 44] = 1e30
    x[8] *= 1e-42
    x[9] = np.finfo(np.float32).min
    u = rng.random(12).astype(np.float32)
    for kw in (dict(), dict(top_k=5), dict(top_p=0.7), dict(min_p=0.2), dict(top_k=100, top_p=0.5, min_p=0.1),
               dict(temperature=0.0), dict(temperature=1e-38), dict(temperature=1e38), dict(temperature=np.inf),
               dict(temperature=np.nan), dict(temperature=-1.0)):
        check(qtts, x, u, **kw)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V", [300, 40000])
def test_min_p_where_many_keys_weigh_the_same(qtts, V, dtype):
    # an infinite temperature makes every finite logit the heaviest; a largest
    # logit of -log(min_p) T puts the border next to zero, where logits are dense
    rng = np.random.default_rng(V)
    x = rng.standard_normal((10, V)).astype(np.float32)
    x[:, ::7] = -np.inf
    x[5:] = np.minimum(x[5:], 0.5) * np.float32(1e-7)
    x[5:, 3] = np.float32(np.log(2.0))
    u = rng.random(10).astype(np.float32)
    T = np.array([np.inf] * 5 + [1.0] * 5, np.float32)
    for m in (0.5, 1.0, 1e-6):
        check(qtts, x, u, temperature=T, min_p=m, dtype=dtype)
        check(qtts, x, u, temperature=T, min_p=m, top_k=20, dtype=dtype)


def test_uniform_numbers_at_the_ends(qtts):
    rng = np.random.default_rng(6)
    u = np.array([0.0, 1.0 - 2.0 ** -24, 1.0, 2.0, -1.0, np.nan, 0.5, 1e-30], np.float32)
    x = (rng.standard_normal((8, 777)) * 2).astype(np.float32)
    x[:, [0, -1]] = -np.inf
    for kw in (dict(), dict(top_k=10), dict(top_p=0.9)):
        tok, kept, _ = run(qtts, torch.from_numpy(x).cuda(), u, **kw)
        for r in range(8):
            wt, wk, _, _ = R.sample(x[r], 1.0, kw.get("top_k", 0), kw.get("top_p", 1.0), 0.0, u[r])
            assert (tok[r], kept[r]) == (wt, wk), (r, kw)


def test_draws_follow_the_weights(qtts):
    # 20000 evenly spread numbers over one row: counts follow the weights to one draw each
    rng = np.random.default_rng(7)
    x = rng.standard_normal(37).astype(np.float32)
    n = 20000
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    rows = torch.from_numpy(x).cuda().repeat(n, 1)
    tok, _, _ = run(qtts, rows, u)
    p = np.exp(x.astype(np.float64) - x.max())
    p /= p.sum()
    assert np.all(np.abs(np.bincount(tok, minlength=37) - n * p) <= 1.0 + n * 2.0 ** -23)


def test_defaults_and_null_outputs_and_many_rows(qtts):
    rng = np.random.default_rng(8)
    x = rng.standard_normal((70000, 9)).astype(np.float32)
    u = rng.random(70000).astype(np.float32)
    dx, du = torch.from_numpy(x).cuda(), torch.from_numpy(u).cuda()
    token = torch.zeros(70000, dtype=torch.int32, device="cuda")
    qtts.sample_rows_dev(dx.data_ptr(), 70000, 9, du.data_ptr(), token.data_ptr())
    w = np.exp(x.astype(np.float64))
    c = np.cumsum(w, 1) / w.sum(1, keepdims=True)
    got = token.cpu().numpy()
    want = np.minimum((c <= u[:, None].astype(np.float64)).sum(1), 8)
    near = np.abs(c - u[:, None]).min(1) < 1e-12
    assert np.all((got == want) | near)


def test_same_rows_same_tokens_whatever_the_batch(qtts):
    rng = np.random.default_rng(9)
    x = torch.from_numpy((rng.standard_normal((160, 20000)) * 2).astype(np.float32)).cuda()
    u = rng.random(160).astype(np.float32)
    kw = dict(temperature=0.9, top_k=300, top_p=0.9)
    a = run(qtts, x, u, **kw)
    for r in (0, 77, 159):
        b = run(qtts, x[r:r + 1], u[r:r + 1], **kw)
        assert all(p[r] == q[0] for p, q in zip(a, b))


def test_in_a_graph_and_on_two_streams_at_once(qtts):
    # no workspace: calls of every path run side by side, and a captured call
    # reads its logits and numbers anew at each replay
    rng = np.random.default_rng(31)
    cases = [(3, 151936, dict(top_p=0.9)), (40, 2048, dict(top_k=50)), (20, 30000, dict(top_k=300, top_p=0.95, min_p=0.01)),
             (2, 151936, dict(temperature=0.0))]
    streams = [torch.cuda.Stream() for _ in range(2)]
    made = []
    for n, V, kw in cases:
        t = {"x": torch.empty(n, V, device="cuda"), "u": torch.empty(n, device="cuda"),
             "token": torch.zeros(n, dtype=torch.int32, device="cuda"), "kept": torch.zeros(n, dtype=torch.int32, device="cuda")}
        t.update({k + "_ptr": torch.full((n,), v, dtype=torch.int32 if k == "top_k" else torch.float32, device="cuda")
                  for k, v in kw.items()})
        made.append((n, V, kw, t))

    def call(n, V, kw, t, stream):
        qtts.sample_rows_dev(t["x"].data_ptr(), n, V, t["u"].data_ptr(), t["token"].data_ptr(), kept_ptr=t["kept"].data_ptr(),
                             stream=stream.cuda_stream, **{k: v.data_ptr() for k, v in t.items() if k.endswith("_ptr")})

    graphs = []
    for i, s in enumerate(streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            for c in made[i::2]:
                call(*c, s)
        graphs.append(g)
    for turn in range(3):
        for n, V, kw, t in made:
            t["x"].copy_(torch.from_numpy((rng.standard_normal((n, V)) * 2.5).astype(np.float32)))
            t["u"].copy_(torch.from_numpy(rng.random(n).astype(np.float32)))
        torch.cuda.synchronize()
        if turn < 2:
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        else:
            for i, c in enumerate(made):
                call(*c, streams[i % 2])
        torch.cuda.synchronize()
        for n, V, kw, t in made:
            x, u = t["x"].cpu().numpy(), t["u"].cpu().numpy()
            for r in range(n):
                wt, wk, _, margin = R.sample(x[r], kw.get("temperature", 1.0), kw.get("top_k", 0),
                                             np.float32(kw.get("top_p", 1.0)), np.float32(kw.get("min_p", 0.0)), u[r])
                assert t["kept"][r].item() == wk
                assert margin <= V * 2.0 ** -45 or t["token"][r].item() == wt


def test_host_logits_are_refused(qtts):
    t = torch.zeros(64)
    d = torch.zeros(64, device="cuda")
    with pytest.raises(qtts.QttsError) as e:
        qtts.sample_rows_dev(t.data_ptr(), 1, 64, d.data_ptr(), d.data_ptr())
    assert e.value.code == qtts.ERR_BADARG
    torch.cuda.synchronize()
