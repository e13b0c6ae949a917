"""A layer of experts and the product's epilogue as far as they go without a GPU: refusals, the table's layout, the oracle's own consistency."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

import mlx_b200
from mlx_b200 import plugin as P
from oracle import moe

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BLOCKS = {"qmatmul_epi": (7, lambda: P.Context.qmm_epi_params(1, 64, 16, 4, 64)), "moe_route": (7, lambda: P.Context.moe_route_params(1, 8, 2)),
          "qmatmul_experts": (8, lambda: P.Context.experts_params(1, 1, 2, 64, 16, 4, 64)), "moe_combine": (5, lambda: P.Context.moe_combine_params(1, 8, 2, 2))}


@pytest.mark.parametrize("name", list(BLOCKS))
def test_null_arguments(name):
    plugin = mlx_b200.Plugin(require_gpu=False)
    n, params = BLOCKS[name]
    for table in (plugin.quant, plugin.short_calls):
        entry = getattr(table, name)
        assert entry(None, None, *[None] * n) == P.ERR_INVALID
        assert entry(None, params(), *[None] * n) == P.ERR_INVALID


@pytest.mark.parametrize("name", list(BLOCKS))
def test_the_compiled_binding_wants_the_right_block(name):
    calls = mlx_b200.Plugin(require_gpu=False).short_calls
    n, _ = BLOCKS[name]
    if not type(calls).__module__.startswith("fastcall"):
        pytest.skip("no compiled binding")
    with pytest.raises(TypeError, match="not a"):
        getattr(calls, name)(None, P.BlockNormParams(), *[None] * n)
    with pytest.raises(TypeError, match="expected"):
        getattr(calls, name)(None, None, *[None] * (n - 1))


def test_header_as_a_c_host_sees_it(tmp_path):
    """The entries are found by the table's size; the parameter blocks have the mirror's layout."""
    kinds = {"lux_qmm_epi_params": P.QmmEpiParams, "lux_moe_route_params": P.MoeRouteParams, "lux_experts_params": P.ExpertsParams,
             "lux_moe_combine_params": P.MoeCombineParams}
    fields = [(c, f[0]) for c, k in kinds.items() for f in k._fields_]
    src = tmp_path / "h.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "lux_cuda_quant.h"\nint main(void) {\n'
                   "    lux_gpu_quant_vtbl t = {0};\n    t.magic = LUX_CUDA_QUANT_MAGIC;\n    t.size = sizeof t;\n"
                   '    printf("%d ", LUX_CUDA_QUANT_HAS(&t, qmatmul_epi) && LUX_CUDA_QUANT_HAS(&t, moe_combine));\n'
                   "    t.size = offsetof(lux_gpu_quant_vtbl, qmatmul_epi);\n"
                   '    printf("%d ", LUX_CUDA_QUANT_HAS(&t, qmatmul_epi) || LUX_CUDA_QUANT_HAS(&t, moe_combine));\n' +
                   "".join(f'    printf("%zu ", sizeof({c}));\n' for c in kinds) +
                   "".join(f'    printf("%zu ", offsetof({c}, {f}));\n' for c, f in fields) + "    return 0;\n}\n")
    exe = tmp_path / "h"
    from mlx_b200 import build
    inc = build.reference_include() or os.path.join(ROOT, "include")
    subprocess.run(["/usr/bin/gcc", "-std=c11", "-Wall", "-Werror", "-I", inc, "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = list(map(int, subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()))
    assert got[:2] == [1, 0]
    assert got[2:] == [C.sizeof(k) for k in kinds.values()] + [getattr(kinds[c], f).offset for c, f in fields]


def test_oracle_route():
    """By hand: ties, masked experts, a token without any, infinities."""
    inf = np.inf
    logits = np.array([[1, 2, 2, 0], [-inf, -inf, 3, -inf], [-inf] * 4, [np.nan, inf, 0, inf], [-0.0, 0.0, -1, -1]])
    ids, w = moe.route(logits, 2)
    assert ids.tolist() == [[1, 2], [2, -1], [-1, -1], [1, 3], [0, 1]]
    np.testing.assert_allclose(w, [[0.5, 0.5], [1, 0], [0, 0], [0.5, 0.5], [0.5, 0.5]])
    ids, w = moe.route(logits[:1], 3, softmax=True, renorm=False, scale=2.0)
    np.testing.assert_allclose(w[0], 2 * np.exp([2, 2, 1]) / np.exp([1, 2, 2, 0]).sum())
    ids, w = moe.route(logits[:1], 2, softmax=False, renorm=False, bias=[1, 0, -inf, 0])
    assert ids.tolist() == [[0, 1]]
    np.testing.assert_allclose(w[0], 1 / (1 + np.exp([-1.0, -2.0])))
    order, pos, offsets = moe.sort(np.array([[1, 0], [-1, 1], [0, 3]]), 4)
    assert order.tolist() == [1, 4, 0, 3, 5] and pos.tolist() == [2, 0, -1, 3, 1, 4] and offsets.tolist() == [0, 2, 4, 4, 5]
