"""CPU tests of the operators on rows chosen by an index: what the entry points refuse,
their host arithmetic, and the shapes that tracing sees."""
import os
import subprocess
import sys

import pytest
import torch

import powersparse_b200 as psb
import powersparse_b200.torch_ops  # noqa: F401  (registers the ops)

INVALID = psb.PS_ERR_INVALID_ARGUMENT
P = 4096  # stands for a device address in calls that are refused before any use of it


def test_names_are_reached_through_the_package():
    for name in ("embedding", "embedding_grad", "route", "route_grad", "dispatch", "dispatch_grad", "combine", "combine_grad",
                 "DispatchPlan", "dispatch_rows"):
        assert name in psb.__all__ and callable(getattr(psb, name)), name
    with pytest.raises(AttributeError):
        psb.no_such_operator


@pytest.mark.parametrize("slots,experts,align", [(0, 1, 1), (0, 8, 128), (1, 1, 1), (5, 3, 4), (7, 2, 128), (100, 64, 16), (64, 64, 3),
                                                 (2**31 - 1, 4, 1)])
def test_dispatch_rows_is_the_largest_fill(slots, experts, align):
    got = psb.dispatch_rows(slots, experts, align)
    # The largest fill: every expert takes one slot more than a multiple of align while slots last.
    full, left = 0, slots
    for _ in range(min(experts, slots)):
        full, left = full + align, left - 1
    assert got == full + left // align * align
    assert got % align == 0 and got >= slots


@pytest.mark.parametrize("args", [(-1, 1, 1), (2**31, 1, 1), (1, 0, 1), (1, 1, 0), (1, 1025, 1), (1, 1, 65537), (1, 2**32 + 1, 1)])
def test_dispatch_rows_refuses(args):
    with pytest.raises(ValueError):
        psb.dispatch_rows(*args)


def test_embedding_grad_workspace_grows_with_the_batch_and_refuses():
    size = psb.load_library().ps_embedding_grad_workspace
    assert 0 <= size(0, 10, 4) <= size(1, 10, 4) <= size(10000, 10, 4) <= size(10000, 100000, 512) < size(1000000, 100000, 512)
    for bad in ((-1, 10, 4), (2**31, 10, 4), (1, 0, 4), (1, 2**31 - 1, 4), (1, 10, 0), (1, 10, 2**24 + 1)):
        assert size(*bad) == -1, bad


def _refused(name, good, **bad):
    """The entry point refuses `good` with each of `bad` in the place of one argument (never called with `good` itself)."""
    lib = psb.load_library()
    for key, value in bad.items():
        for v in value if isinstance(value, list) else [value]:
            args = dict(good)
            assert key in args, key
            args[key] = v
            assert getattr(lib, name)(*args.values()) == INVALID, (name, key, v)
            assert lib.ps_last_error().startswith(name.encode()), (name, key, v)


def test_c_entry_points_refuse():
    big = 2**24 + 1
    _refused("ps_embedding", dict(table=P, dtype=1, rows=10, width=8, table_stride=8, tokens=P, index_type=0, n=4, scale=1.0, out=P,
                                  out_stride=8, stream=None),
             table=[None, P + 1], dtype=[-1, 3], rows=[0, -1], width=[0, -1, big], table_stride=[7, 2**40], tokens=[None, P + 2],
             index_type=[-1, 2], n=[-1, 2**31], out=[None, P + 1], out_stride=7)
    _refused("ps_embedding_grad", dict(grad=P, grad_dtype=1, grad_stride=8, tokens=P, index_type=1, n=4000, scale=1.0, padding=-1,
                                       accumulate=0, grad_table=P, table_dtype=0, table_stride=8, rows=10, width=8, workspace=P,
                                       workspace_bytes=1 << 30, stream=None),
             grad=[None, P + 1], grad_dtype=[5, -1], grad_stride=7, tokens=[None, P + 4], index_type=2, n=[-1, 2**31],
             grad_table=[None, P + 2], table_dtype=[2, 9], table_stride=7, rows=[0, 2**31 - 1], width=[0, big],
             workspace=[None, P + 128], workspace_bytes=[0, 1000])
    _refused("ps_route", dict(logits=P, dtype=0, stride=8, tokens=4, experts=8, top_k=2, normalize=1, weights=P, chosen=P, stream=None),
             logits=[None, P + 2], dtype=3, stride=7, tokens=-1, experts=[0, 1025, 1], top_k=[0, 9, 33], weights=[None, P + 1],
             chosen=[None, P + 1])
    _refused("ps_route_grad", dict(grad=P, logits=P, dtype=0, stride=8, weights=P, chosen=P, tokens=4, experts=8, top_k=2, normalize=0,
                                   out=P, out_stride=8, stream=None),
             grad=[None, P + 1], logits=None, dtype=3, stride=7, weights=None, chosen=None, tokens=-1, experts=[0, 1025],
             top_k=[0, 9], out=[None, P + 2], out_stride=7)
    _refused("ps_dispatch", dict(x=P, dtype=1, x_stride=8, chosen=P, index_type=0, tokens=4, top_k=2, experts=8, align=1, width=8,
                                 rows=P, rows_stride=8, row_count=8, zero_tail=0, position=P, offsets=P, counts=P, stream=None),
             x=[None, P + 1], dtype=-1, x_stride=7, chosen=[None, P + 1], index_type=2, tokens=[-1, 2**31 - 1], top_k=[0, 33],
             experts=[0, 1025], align=[0, 65537, 2], width=[0, big], rows=[None, P + 1], rows_stride=7, row_count=[7, -1],
             position=None, offsets=None, counts=None)
    _refused("ps_combine", dict(y=P, dtype=0, y_stride=8, row_count=8, position=P, weights=P, add=P, add_stride=8, tokens=4, top_k=2,
                                width=8, out=P, out_stride=8, stream=None),
             y=[None, P + 2], dtype=3, y_stride=7, row_count=-1, position=[None, P + 2], weights=P + 2, add=P + 1, add_stride=7,
             tokens=-1, top_k=[0, 33], width=[0, big], out=[None, P + 2], out_stride=7)
    _refused("ps_combine_grad", dict(grad=P, dtype=2, grad_stride=8, y=P, y_stride=8, row_count=8, position=P, offsets=P, counts=P,
                                     experts=4, weights=P, tokens=4, top_k=2, width=8, grad_y=P, grad_y_stride=8, zero_tail=1,
                                     grad_weights=P, stream=None),
             grad=[None, P + 1], dtype=3, grad_stride=7, y=[None, P + 1], y_stride=7, row_count=-1, position=None, offsets=None,
             counts=None, experts=[0, 1025], weights=None, tokens=-1, top_k=[0, 33], width=0, grad_y=None, grad_y_stride=7,
             grad_weights=None)


def test_python_functions_refuse_host_tensors():
    x, i = torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int32)
    plan = psb.DispatchPlan(i, torch.zeros(5, dtype=torch.int32), torch.zeros(4, dtype=torch.int32))
    for call in (lambda: psb.embedding(x, i), lambda: psb.embedding_grad(x, i[:, 0], 4), lambda: psb.route(x, 2),
                 lambda: psb.route_grad(x[:, :2], x, x[:, :2], i), lambda: psb.dispatch(x, i, 4), lambda: psb.combine(x, plan),
                 lambda: psb.combine_grad(x, x, plan, x[:, :2]), lambda: psb.embedding(None, i)):
        with pytest.raises(ValueError, match="CUDA tensor"):
            call()


def test_ops_are_registered_and_traced_on_meta_tensors():
    ops = torch.ops.powersparse
    table, tokens = torch.empty(100, 16, device="meta", dtype=torch.bfloat16), torch.empty(3, 5, device="meta", dtype=torch.int64)
    assert ops.embedding(table, tokens).shape == (3, 5, 16)
    assert ops.embedding_grad(torch.empty(3, 5, 16, device="meta"), tokens, 100).shape == (100, 16)
    weights, chosen = ops.route(torch.empty(7, 12, device="meta", dtype=torch.float16), 3)
    assert weights.shape == chosen.shape == (7, 3) and weights.dtype == torch.float32 and chosen.dtype == torch.int32
    x = torch.empty(7, 16, device="meta")
    rows, position, offsets, counts = ops.dispatch(x, chosen, 12, 4)
    assert rows.shape == (psb.dispatch_rows(21, 12, 4), 16) and position.shape == (7, 3)
    assert offsets.shape == (13,) and counts.shape == (12,)
    assert ops.combine(rows, position, offsets, counts, weights, x).shape == (7, 16)
    grad_y, grad_w = ops.combine_grad(x, rows, position, offsets, counts, weights)
    assert grad_y.shape == rows.shape and grad_w.shape == weights.shape


@pytest.mark.parametrize("args", [(-1, 1, 1), (2**31, 1, 1), (1, 0, 1), (1, -1, 1), (1, 1, 0), (1, 1025, 1), (1, 1, 65537), (1, 1, -1)])
def test_c_dispatch_rows_refuses_what_dispatch_refuses(args):
    assert psb.load_library().ps_dispatch_rows(*args) == -1


def test_c_dispatch_rows_takes_the_largest_arguments():
    assert psb.load_library().ps_dispatch_rows(1, 1024, 65536) == 65536


def _without_torch(code):
    """Runs `code` in a process in which `import torch` fails as where torch is not installed."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, "-c", "import sys\nsys.modules['torch'] = None\n" + code], capture_output=True, text=True,
                         timeout=600, cwd=root)
    assert run.returncode == 0, run.stdout + run.stderr
    return run.stdout


def test_star_import_without_torch():
    _without_torch("from powersparse_b200 import *\n"
                   "assert callable(SpMM) and PS_OK == 0\n"
                   "assert 'embedding' not in globals()")


def test_build_without_torch(tmp_path):
    """The libraries and the command line tools build; the module on torch tensors is left out."""
    _without_torch("from powersparse_b200 import build\n"
                   f"build.ROWS_MODULE = {str(tmp_path / '_rows.so')!r}\n"
                   "build.build_all()")
    assert not list(tmp_path.iterdir())


def test_a_module_of_another_torch_is_built_again_and_not_loaded(tmp_path, monkeypatch):
    from powersparse_b200 import build, rows
    module = tmp_path / "_rows.so"
    built = []

    def fake(cmd):
        built.append(cmd)
        module.write_bytes(b"")
    monkeypatch.setattr(build, "ROWS_MODULE", str(module))
    monkeypatch.setattr(build, "_run", fake)
    build.build_rows_module()
    build.build_rows_module()
    assert len(built) == 1  # fresh
    record = tmp_path / "_rows.so.built_for"
    assert torch.__version__ in record.read_text()
    record.write_text("torch 1.0, cpython-38")
    monkeypatch.setattr(rows, "_MODULE_PATH", str(module))
    monkeypatch.setattr(rows, "_BUILT_FOR_PATH", str(record))
    with pytest.raises(RuntimeError, match="torch 1.0"):
        rows._load_native()
    build.build_rows_module()
    assert len(built) == 2 and torch.__version__ in record.read_text()
    record.unlink()  # of unknown origin
    build.build_rows_module()
    assert len(built) == 3


def test_embedding_op_refuses_a_padding_outside_the_table_in_the_forward_pass():
    table, tokens = torch.empty(100, 16, device="meta"), torch.empty(5, device="meta", dtype=torch.int64)
    for padding in (-1, 100, 2**40):
        with pytest.raises(ValueError, match="padding"):
            torch.ops.powersparse.embedding(table, tokens, 1.0, padding)
    for padding in (None, 0, 99):
        assert torch.ops.powersparse.embedding(table, tokens, 1.0, padding).shape == (5, 16)


def test_embedding_grad_of_few_tokens_in_wide_rows_is_sorted():
    """The one launch for few tokens (no workspace) adds up a token's rows in few blocks: not for more than 5 * 2^20 elements."""
    size = psb.load_library().ps_embedding_grad_workspace
    for n, width in ((2048, 2560), (1024, 5120), (1, 5 * 2**20), (2047, 2560), (0, 2**24)):
        assert size(n, 4096, width) == 0, (n, width)
    for n, width in ((2048, 2561), (2048, 8192), (1025, 5120), (1, 5 * 2**20 + 1), (2049, 1)):
        assert size(n, 4096, width) > 0, (n, width)
