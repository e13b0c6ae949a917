"""The Python binding of the entries that a table may or may not have, without a GPU."""
import ctypes as C
from types import SimpleNamespace

import pytest

from mlx_b200 import plugin as P

CALLS = {"mx4_quantize": lambda c, b: c.mx4_quantize(b, b, b, 1, 32, 1, P.F32), "mx4_dequantize": lambda c, b: c.mx4_dequantize(b, b, b, 1, 32, 1, P.F32),
         "mx4_matmul": lambda c, b: c.mx4_matmul(b, b, b, b, b, 1, 32, 1, 1, P.F32),
         "block_norm": lambda c, b: c.block_norm(c.block_norm_params(1, 32), b, None, None, None, None, None, None, b, None),
         "mx4_scale_bytes": lambda c, b: c.mx4_scale_bytes(1, 32, 1)}


@pytest.fixture()
def table():
    """A table whose entries behind version 7's last note that they were called, and a plugin around it."""
    called = []
    t = P.QuantVtbl(magic=P.QUANT_MAGIC)
    for name, kind in P.QuantVtbl._fields_:
        if name in CALLS:
            setattr(t, name, kind(lambda *a, name=name: called.append(name) or 0))
    plugin = SimpleNamespace(quant=t, vtbl=SimpleNamespace(create_context=lambda device: 1, destroy_context=lambda handle: None), short_calls=t, last_error=lambda: "")
    plugin.check = lambda code, what: P.Plugin.check(plugin, code, what)
    return t, plugin, called


@pytest.mark.parametrize("last", [None] + list(CALLS))
def test_entries_past_the_end_of_the_table_are_not_called(table, last):
    """Nor kept: what lies behind a shorter table is no function.  Whole tables and tables that end behind `last`, or ahead of all five."""
    t, plugin, called = table
    names = [n for n, _ in P.QuantVtbl._fields_ if n in CALLS]
    there = names[:names.index(last) + 1] if last else []
    end = getattr(P.QuantVtbl, there[-1] if there else names[0])
    t.size = end.offset + (end.size if there else 0)
    ctx = P.Context(plugin)
    for name in names:
        del called[:]
        if name in there:
            CALLS[name](ctx, SimpleNamespace(handle=1))
            assert called == [name]
        else:
            with pytest.raises(P.BackendError) as e:
                CALLS[name](ctx, SimpleNamespace(handle=1))
            assert e.value.code == P.ERR_NOT_SUPPORTED and name in str(e.value) and not called


@pytest.mark.parametrize("compiler", ["fails", "is not there"])
def test_a_build_without_the_compiled_binding(monkeypatch, tmp_path, compiler):
    """The compiled binding is an extra: where it cannot be built the build goes on, none of an earlier build stays, and the calls go through ctypes."""
    import subprocess

    from mlx_b200 import build
    path = tmp_path / "fastcall.so"
    path.write_bytes(b"an earlier build's")
    monkeypatch.setattr(build, "FASTCALL_PATH", str(path))
    commands = []

    def run(cmd, **kw):
        commands.append(cmd)
        if compiler == "fails":
            raise subprocess.CalledProcessError(1, cmd)
        raise FileNotFoundError(cmd[0])
    monkeypatch.setattr(build.subprocess, "run", run)
    monkeypatch.setattr(build.os.path, "exists", lambda p, exists=build.os.path.exists: p.endswith("Python.h") or exists(p))
    build.build_fastcall("include", force=True)
    assert len(commands) == 1 and not path.exists()
    t = P.QuantVtbl(magic=P.QUANT_MAGIC, size=C.sizeof(P.QuantVtbl))
    assert P._short_calls(t) is t


@pytest.mark.parametrize("kind", ["int32", "int64", "uint64"])
def test_sizes_that_are_numpy_integers(kind):
    """As with ctypes: whatever Python takes for an index is a size, floats are not."""
    import numpy as np

    import mlx_b200
    plugin = mlx_b200.Plugin(require_gpu=False)
    T = getattr(np, kind)
    for table in (plugin.quant, plugin.short_calls):
        assert table.mx4_quantize(None, None, None, None, T(1), T(32), T(32), T(1), T(P.F32), np.float32(1)) == P.ERR_INVALID
        assert table.mx4_matmul(None, None, None, None, None, None, T(1), T(32), T(1), T(1), T(P.F32), np.float32(1)) == P.ERR_INVALID
        with pytest.raises((TypeError, C.ArgumentError)):
            table.mx4_quantize(None, None, None, None, 1, 32, 32.0, 1, P.F32, 1.0)
