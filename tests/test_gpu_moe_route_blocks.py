"""The router around the borders of its launches: one block with a token a warp and with two, the fewest tokens of several blocks; given experts in more slots than there are experts."""
import numpy as np
import pytest

from mlx_b200 import F32
from mlx_b200 import plugin as P
from oracle import moe
from test_gpu_moe_route import check, check_sort, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [16, 17, 31, 32, 33])
@pytest.mark.parametrize("E,k", [(256, 8), (257, 1), (300, 6), (1024, 32)])
@pytest.mark.parametrize("with_bias", [False, True])
def test_tokens_of_one_block(ctx, T, E, k, with_bias):
    rng = np.random.default_rng(T + E)
    v = (rng.standard_normal((T, E)) * 2).astype(np.float32)
    v[T // 2] = -np.inf
    bias = (rng.standard_normal(E) * 0.1).astype(np.float32) if with_bias else None
    score = P.SCORE_SIGMOID if with_bias else P.SCORE_SOFTMAX
    got = run(ctx, ctx.moe_route_params(T, E, k, score=score, logits_dtype=F32), ctx.upload(v), ctx.upload(bias) if with_bias else None, T, k, E)
    check(got, moe.route(v, k, not with_bias, True, 1.0, bias), T, k, E)


@pytest.mark.parametrize("T", [1, 20, 32, 33, 700])
@pytest.mark.parametrize("E,k", [(1, 32), (3, 32), (1024, 2)])
def test_given_experts(ctx, T, E, k):
    ids = np.random.default_rng(T).integers(-1, E + 1, (T, k)).astype(np.int32)
    got = run(ctx, ctx.moe_route_params(T, E, k), None, None, T, k, E, ids=ids)
    check_sort(got, np.where((ids >= 0) & (ids < E), ids, -1), E)
