"""router_topk by scores, with a bias and groups, against the 64-bit oracle: the routes are equal, the weights within two roundings (2^-23; sums and quotients are 64 bits wide)."""
import numpy as np
import pytest
import torch

from oracle import mxfp4 as orc
from tests.gpu_util import dev, host, kernel

pytestmark = pytest.mark.gpu


def run(logits, top_k, bias=None, renormalize=True, rows=None, **options):
    m, experts = logits.shape
    ids = torch.full((m, top_k), -7, dtype=torch.int32, device="cuda")
    prob = torch.full((m, top_k), -7.0, device="cuda")
    named = dict(IDs=ids, Logits=dev(logits.astype(np.float32)), Prob=prob)
    if bias is not None:
        named["Bias"] = dev(np.asarray(bias, np.float32))
    if rows is not None:
        named["m"] = rows
    kernel("router_topk", M=m, E=experts, top_k=top_k, renormalize=renormalize, bias=bias is not None, dynamic_rows=rows is not None, **options)(**named)
    return host(ids), host(prob)


def check(logits, top_k, bias=None, renormalize=True, **options):
    logits = logits.astype(np.float32)
    bias = None if bias is None else np.asarray(bias, np.float32)
    ids, prob = run(logits, top_k, bias, renormalize, **options)
    scale = {"scale": float(np.float32(options["scale"]))} if "scale" in options else {}
    want_ids, want = orc.routes(logits, top_k, bias=bias, renormalize=renormalize, **dict(options, **scale))
    np.testing.assert_array_equal(ids, want_ids)
    np.testing.assert_allclose(prob, want, rtol=2.0**-23, atol=2.0**-149)
    return ids, prob


@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
@pytest.mark.parametrize("m,experts,top_k,groups,top_groups", [(1, 8, 2, 1, 1), (3, 60, 6, 1, 1), (5, 128, 8, 1, 1), (33, 256, 8, 8, 4), (17, 160, 6, 8, 3), (9, 64, 1, 64, 1),
                                                               (7, 512, 10, 16, 5), (6, 1000, 64, 4, 2), (4, 1024, 16, 2, 1), (2, 1, 1, 1, 1), (70, 96, 4, 3, 2), (3, 64, 64, 1, 1)])
def test_routes_and_weights(scoring, m, experts, top_k, groups, top_groups):
    rng = np.random.default_rng(m * experts + top_k)
    logits = rng.standard_normal((m, experts)) * 2
    bias = rng.standard_normal(experts) * (0.1 if scoring == "sigmoid" else 0.01)
    for best in (1, 2):
        check(logits, top_k, bias, scoring=scoring, groups=groups, top_groups=top_groups, group_best=best)
    check(logits, top_k, bias, renormalize=False, scoring=scoring, groups=groups, top_groups=top_groups, scale=2.5)
    check(logits, top_k, scoring=scoring, groups=groups, top_groups=top_groups, scale=0.1)


def test_scores_that_32_bits_do_not_tell_apart():
    rng = np.random.default_rng(5)
    # logits a last place apart around values where the sigmoid is flat, and biases that put other experts beside them
    logits = np.full((200, 64), 9.0, np.float32)
    for _ in range(6):
        logits = np.where(rng.random(logits.shape) < 0.5, np.nextafter(logits, np.float32(99)), logits)
    check(logits, 8, scoring="sigmoid", groups=8, top_groups=4)
    check(logits, 8, np.zeros(64), scoring="softmax")
    # as many pairs whose sums of score and bias differ in the 40th bit
    base = rng.standard_normal((100, 32)).astype(np.float32)
    bias = np.zeros(64, np.float32)
    bias[32:] = 0.25
    score = 1 / (1 + np.exp(-base.astype(np.float64)))
    with np.errstate(all="ignore"):
        other = -np.log(1 / (score - 0.25) - 1)
    logits = np.concatenate([base, np.nan_to_num(other, nan=-3.0, posinf=-3.0, neginf=-3.0)], 1)
    check(logits, 12, bias, scoring="sigmoid")
    check(logits, 12, bias, scoring="sigmoid", groups=16, top_groups=6)


def test_ties_go_to_the_lower_id_and_the_lower_group():
    logits = np.zeros((3, 96))
    ids, _ = check(logits, 5, scoring="sigmoid", groups=8, top_groups=2)
    assert (ids == np.arange(5)).all()
    logits[:, 40:] = 1
    ids, _ = check(logits, 5, scoring="sigmoid", groups=8, top_groups=2)
    assert (ids == np.arange(40, 45)).all()  # the group of 36 to 47 has two of them, as any behind it, and comes first


@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
def test_closed_experts_and_scores_of_nothing(scoring):
    rng = np.random.default_rng(6)
    logits = rng.standard_normal((6, 32))
    bias = np.zeros(32)
    bias[rng.permutation(32)[:28]] = -np.inf       # four experts left for six routes
    _, prob = check(logits, 6, bias, scoring=scoring)
    assert (prob[:, 4:] == 0).all() and (prob[:, :4] > 0).all()
    check(logits, 6, bias, scoring=scoring, groups=8, top_groups=3)
    _, prob = check(logits, 3, np.full(32, -np.inf), scoring=scoring, groups=4, top_groups=2)
    assert (prob == 0).all()
    bias = np.zeros(32)
    bias[[3, 20]] = np.inf                         # always chosen
    bias[7] = np.nan                               # never before others
    ids, _ = check(logits, 4, bias, scoring=scoring)
    assert (ids[:, :2] == [3, 20]).all()
    check(logits, 4, bias, scoring=scoring, groups=8, top_groups=3)


@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
def test_logits_of_nan_and_infinity(scoring):
    rng = np.random.default_rng(7)
    logits = rng.standard_normal((6, 40))
    logits[0, 5] = np.nan
    logits[1, :] = np.nan
    logits[2, 7] = np.inf
    logits[3, :] = -np.inf
    logits[4, 3:] = -np.inf
    logits[5] = -800
    ids, prob = check(logits, 5, np.zeros(40), scoring=scoring)
    assert not np.isnan(prob).any() and all(len(set(row)) == 5 for row in ids.tolist())
    check(logits, 5, scoring=scoring, groups=8, top_groups=2)


def test_fewer_rows_than_the_capacity_leave_the_rest():
    logits = np.random.default_rng(8).standard_normal((9, 64))
    ids, prob = run(logits, 4, rows=5, scoring="sigmoid")
    want, weights = orc.routes(logits.astype(np.float32)[:5], 4, scoring="sigmoid")
    np.testing.assert_array_equal(ids[:5], want)
    np.testing.assert_allclose(prob[:5], weights, rtol=2.0**-23)
    assert (ids[5:] == -7).all() and (prob[5:] == -7).all()


def test_captured_and_replayed():
    logits = torch.randn((37, 160), device="cuda")
    bias = torch.randn(160, device="cuda") * 0.1
    ids, prob = torch.empty((37, 6), dtype=torch.int32, device="cuda"), torch.empty((37, 6), device="cuda")
    router = kernel("router_topk", M=37, E=160, top_k=6, scoring="sigmoid", bias=True, groups=8, top_groups=3, scale=2.5)
    torch.cuda.synchronize()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        router(stream=stream.cuda_stream, Bias=bias, IDs=ids, Logits=logits, Prob=prob)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        want_ids, want = orc.routes(host(logits), 6, scoring="sigmoid", bias=host(bias), groups=8, top_groups=3, scale=2.5)
        np.testing.assert_array_equal(host(ids), want_ids)
        np.testing.assert_allclose(host(prob), want, rtol=2.0**-23, atol=2.0**-149)
        logits.copy_(logits.roll(1, 1))
        bias.neg_()
        torch.cuda.synchronize()
