"""cb200_moe_route against the plain definition in 64 bits: ids equal, weights within what 32-bit arithmetic allows."""
import numpy as np
import pytest

import moe_reference as R

pytestmark = pytest.mark.gpu

# A weight is a score, renormalised or not.  sigmoid: 2^-20.9 relative; softmax: 44 * 2^-24 from expf, the sum of up to
# 1024 terms and the quotient, and |x - max| * 2^-24 from the difference, |x - max| <= 100 for every weight compared
# here: together below 2^-16.8.  Renormalising divides by a sum with errors of the same signs and size.
RTOL = 2.0 ** -16


def call(torch, capi, logits, top_k, bias=None, pitch=0, count=None, stream=None, experts=None, **kw):
    t, e = logits.shape[0], experts or logits.shape[1]
    types = {torch.float32: capi.DTYPE_F32, torch.bfloat16: capi.DTYPE_BF16, torch.float16: capi.DTYPE_F16}
    w = torch.full((t, top_k), -7.0, device=logits.device)
    ids = torch.full((t, top_k), -7, dtype=torch.int32, device=logits.device)
    capi.moe_route(logits, w, ids, t, e, top_k, bias=bias, logits_type=types[logits.dtype], logits_pitch=pitch,
                   token_count=count, stream=stream, **kw)
    return w, ids


def check(w, ids, want_ids, want_w):
    assert np.array_equal(ids.cpu().numpy(), want_ids)
    got = w.cpu().numpy().astype(np.float64)
    assert (np.abs(got - want_w) <= RTOL * np.abs(want_w) + 1e-37).all(), np.abs(got / np.where(want_w, want_w, 1) - 1).max()


@pytest.mark.parametrize("t,e,k,groups,kept", [
    (1, 1, 1, 1, 1), (1, 256, 8, 8, 4), (5, 7, 3, 1, 1), (33, 60, 4, 1, 1), (64, 64, 6, 8, 3), (130, 96, 8, 3, 2),
    (7, 160, 6, 8, 3), (40, 256, 8, 8, 4), (9, 384, 8, 1, 1), (3, 1024, 32, 32, 5), (6, 40, 10, 20, 5), (12, 33, 32, 1, 1),
    (5, 31, 31, 31, 31),
])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_route_matches_the_definition(cuda, t, e, k, groups, kept, dtype):
    import torch
    from catlass_b200 import capi
    g = torch.Generator(device="cuda").manual_seed(t * 1000 + e)
    logits = (1.5 * torch.randn((t, e), generator=g, device=cuda)).to(getattr(torch, dtype))
    bias = 0.1 * torch.randn((e,), generator=g, device=cuda)
    x, b = logits.double().cpu().numpy(), bias.double().cpu().numpy()
    for sigmoid in (False, True):
        for with_bias in (False, True):
            for top2 in (False, True):
                renorm = sigmoid != top2
                w, ids = call(torch, capi, logits, k, bias=bias if with_bias else None, groups=groups, groups_kept=kept,
                              score=capi.ROUTE_SIGMOID if sigmoid else capi.ROUTE_SOFTMAX, renormalize=renorm, scaling=2.5,
                              group_score=capi.ROUTE_GROUP_TOP2_SUM if top2 else capi.ROUTE_GROUP_MAX)
                check(w, ids, *R.route(x, k, sigmoid, b if with_bias else None, groups, kept, top2, renorm, 2.5))


def test_route_many_tokens(cuda):
    """Enough tokens that some have keys closer than 32 bits tell apart."""
    import torch
    from catlass_b200 import capi
    g = torch.Generator(device="cuda").manual_seed(3)
    logits = (1.5 * torch.randn((20011, 256), generator=g, device=cuda)).to(torch.bfloat16)
    bias = 0.1 * torch.randn((256,), generator=g, device=cuda)
    for sigmoid, bb in ((True, bias), (False, bias), (True, torch.zeros_like(bias)), (False, None)):
        w, ids = call(torch, capi, logits, 8, bias=bb, groups=8, groups_kept=4, group_score=capi.ROUTE_GROUP_TOP2_SUM,
                      score=capi.ROUTE_SIGMOID if sigmoid else capi.ROUTE_SOFTMAX)
        check(w, ids, *R.route(logits.double().cpu().numpy(), 8, sigmoid,
                               None if bb is None else bb.double().cpu().numpy(), 8, 4, True, True))


@pytest.mark.parametrize("e,k,groups,kept", [(17, 8, 1, 1), (60, 4, 1, 1), (64, 8, 8, 3), (64, 1, 4, 2), (96, 6, 3, 1),
                                             (128, 8, 8, 8), (128, 7, 4, 2), (200, 5, 1, 1), (256, 8, 4, 2), (256, 8, 8, 1)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_route_batches_with_holes_and_ties(cuda, e, k, groups, kept, dtype):
    """Batches that share warps among tokens: coarse logits (many equal), masked ones, whole rows and groups of them, and
    biases that bring different logits to within 1e-7 of one another."""
    import torch
    from catlass_b200 import capi
    t = 4103
    rng = np.random.default_rng(e + k)
    x = (1.5 * rng.standard_normal((t, e))).astype(np.float32)
    x[::3] = np.round(x[::3] * 4) / 4
    x[1::7][rng.random((len(x[1::7]), e)) < 0.7] = -np.inf
    x[5::11, : e // groups] = np.nan
    x[40] = -np.inf
    x[41, 1:] = -np.inf
    logits = torch.from_numpy(x).to(cuda).to(getattr(torch, dtype))
    x = logits.double().cpu().numpy()
    with np.errstate(over="ignore"):
        s = 1 / (1 + np.exp(-np.nan_to_num(x[0], nan=0.0)))
    biases = [None, np.zeros(e, np.float32), (0.1 * rng.standard_normal(e)).astype(np.float32), (0.9 - s).astype(np.float32)]
    for sigmoid in (True, False):
        for bias in biases:
            for top2 in (True, False):
                w, ids = call(torch, capi, logits, k, bias=None if bias is None else torch.from_numpy(bias).to(cuda),
                              groups=groups, groups_kept=kept, renormalize=top2,
                              score=capi.ROUTE_SIGMOID if sigmoid else capi.ROUTE_SOFTMAX,
                              group_score=capi.ROUTE_GROUP_TOP2_SUM if top2 else capi.ROUTE_GROUP_MAX)
                check(w, ids, *R.route(x, k, sigmoid, bias, groups, kept, top2, top2))


def test_route_ties_and_near_ties(cuda):
    import torch
    from catlass_b200 import capi
    # all equal: the lowest indices, of groups and of experts
    logits = torch.zeros((3, 64), device=cuda)
    for bias in (None, torch.full((64,), 0.25, device=cuda)):
        _, ids = call(torch, capi, logits, 6, bias=bias, groups=4, groups_kept=2, group_score=capi.ROUTE_GROUP_TOP2_SUM,
                      score=capi.ROUTE_SIGMOID)
        assert np.array_equal(ids.cpu().numpy(), np.tile(np.arange(6), (3, 1)))
    # -0 and +0 are the same logit
    logits = torch.zeros((1, 8), device=cuda)
    logits[0, 0] = -0.0
    assert call(torch, capi, logits, 2)[1].tolist() == [[0, 1]]
    # keys that differ by about 1e-8 only: sigmoid(x) + bias with a bias that nearly makes up for the difference
    rng = np.random.default_rng(5)
    x = rng.uniform(-3, 3, (64, 16)).astype(np.float32)
    s = 1 / (1 + np.exp(-x[0].astype(np.float64)))
    bias = (1.0 - s).astype(np.float32)         # every key of row 0 is 1 up to the rounding of the bias
    x[1:] = x[0] + rng.choice([0, 2.0 ** -22, -2.0 ** -22], (63, 16)).astype(np.float32)
    w, ids = call(torch, capi, torch.from_numpy(x).to(cuda), 5, bias=torch.from_numpy(bias).to(cuda),
                  score=capi.ROUTE_SIGMOID)
    check(w, ids, *R.route(x, 5, True, bias, renormalize=True))
    w, ids = call(torch, capi, torch.from_numpy(x).to(cuda), 5, bias=torch.from_numpy(bias).to(cuda), groups=4, groups_kept=2,
                  score=capi.ROUTE_SIGMOID, group_score=capi.ROUTE_GROUP_TOP2_SUM)
    check(w, ids, *R.route(x, 5, True, bias, 4, 2, True, True))


def test_route_masked_logits(cuda):
    """-inf and NaN cannot be chosen, rows that have nothing left, logits of +inf, values at the ends of the range."""
    import torch
    from catlass_b200 import capi
    inf, nan = float("inf"), float("nan")
    x = np.random.default_rng(1).standard_normal((9, 48)).astype(np.float32)
    x[0, :] = -inf
    x[1, :] = nan
    x[2, 5:] = -inf
    x[3, ::2] = nan
    x[4, 7] = inf
    x[5, [3, 9]] = inf
    x[6, :] = np.finfo(np.float32).min
    x[6, 4] = np.finfo(np.float32).max
    x[7, :16] = -inf                      # a whole group
    x[8, :] = -80.0                       # sigmoids near the bottom of the normal range
    x[8, 11] = -75.0
    bias = np.linspace(-0.2, 0.2, 48).astype(np.float32)
    for sigmoid in (False, True):
        for b in (None, bias):
            for groups, kept, top2 in ((1, 1, False), (3, 1, True), (3, 2, False), (24, 4, True)):
                for renorm in (False, True):
                    w, ids = call(torch, capi, torch.from_numpy(x).to(cuda), 8, groups=groups, groups_kept=kept,
                                  bias=None if b is None else torch.from_numpy(b).to(cuda), renormalize=renorm,
                                  score=capi.ROUTE_SIGMOID if sigmoid else capi.ROUTE_SOFTMAX,
                                  group_score=capi.ROUTE_GROUP_TOP2_SUM if top2 else capi.ROUTE_GROUP_MAX)
                    check(w, ids, *R.route(x, 8, sigmoid, b, groups, kept, top2, renorm))


def test_route_strided_padded_and_other_stream(cuda):
    import torch
    from catlass_b200 import capi
    g = torch.Generator(device="cuda").manual_seed(8)
    wide = torch.randn((50, 101), generator=g, device=cuda).to(torch.bfloat16)
    part = wide[:, 3:67]                                     # rows 101 apart, starting at an odd element
    want = R.route(part.double().cpu().numpy(), 4, False, renormalize=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    count = torch.tensor([20], dtype=torch.int32, device=cuda)
    w, ids = call(torch, capi, part, 4, pitch=101, stream=side)
    w2, ids2 = call(torch, capi, part, 4, pitch=101, count=count, stream=side)
    torch.cuda.synchronize()
    check(w, ids, *want)
    check(w2[:20], ids2[:20], want[0][:20], want[1][:20])
    assert (ids2[20:] == -1).all() and (w2[20:] == 0).all()
    for n, filled in ((-3, 0), (0, 0), (1 << 30, 50)):
        count.fill_(n)
        _, ids3 = call(torch, capi, part, 4, pitch=101, count=count)
        assert int((ids3 >= 0).all(1).sum()) == filled


def test_route_in_a_graph(cuda):
    import torch
    from catlass_b200 import capi
    logits = torch.randn((17, 128), device=cuda)
    w = torch.empty((17, 4), device=cuda)
    ids = torch.empty((17, 4), dtype=torch.int32, device=cuda)
    capi.moe_route(logits, w, ids, 17, 128, 4)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        capi.moe_route(logits, w, ids, 17, 128, 4)
    for seed in (1, 2):
        logits.copy_(torch.randn((17, 128), generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        check(w, ids, *R.route(logits.double().cpu().numpy(), 4, False, renormalize=True))


def test_route_empty_batch_and_short_buffers(cuda):
    import torch
    from catlass_b200 import capi
    before = capi.launch_count()
    call(torch, capi, torch.empty((0, 64), device=cuda), 4)
    assert capi.launch_count() == before
    x = torch.zeros((4, 64), device=cuda)
    w, ids = torch.zeros((4, 4), device=cuda), torch.zeros((4, 4), dtype=torch.int32, device=cuda)
    with pytest.raises(ValueError):
        capi.moe_route(x, w, ids, 5, 64, 4)
    with pytest.raises(ValueError):
        capi.moe_route(x, w, ids, 4, 64, 5)
    with pytest.raises(ValueError):
        capi.moe_route(x, w, ids, 4, 64, 4, logits_pitch=65)
    with pytest.raises(capi.CallError):
        capi.moe_route(x, w, ids, 4, 64, 4, groups=3)
