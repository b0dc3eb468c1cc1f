"""The forms that the block's norms choose by row count, width and types,
against the formulas in 64 bits; tolerances as in test_gpu_block_norms.py."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover - collected on CPU hosts too
    pytest.skip("needs a CUDA device", allow_module_level=True)

from test_gpu_block_norms import BF16, DEV, F16, F32, check, make, reference  # noqa: E402

from dispatch_b200 import _lib as L  # noqa: E402
from dispatch_b200.kernels.block import norm_gate_residual, norm_gate_residual_backward, rms_norm  # noqa: E402

SMS = torch.cuda.get_device_properties(0).multi_processor_count


@pytest.fixture(autouse=True)
def _device_status_clean():
    yield
    L.check_device_status(DEV)


def run(t, h, dtypes, gate, norm_dtype, a=0.7, eps=1e-6, seed=0):
    """Forward and backward, normed and its gradient in norm_dtype."""
    i = make(t, h, dtypes, gate, seed=seed)
    dn = i["d_normed"].to(norm_dtype)
    args = (i["y"], i["residual"], i["post_weight"], i["next_weight"])
    kw = dict(gate=i["gate"], residual_scale=a, eps=eps)
    a32, e32 = (torch.tensor(v, dtype=F32).item() for v in (a, eps))
    want = reference(*args, i["gate"], a32, e32, i["d_out"], dn)
    out, normed = norm_gate_residual(*args, norm_dtype=norm_dtype, **kw)
    assert normed.dtype == norm_dtype
    check("out", out, want["out"])
    check("normed", normed, want["normed"])
    grads = norm_gate_residual_backward(i["d_out"], dn, *args, **kw)
    for name, got in zip(("dy", "dresidual", "dpost", "dnext", "dgate"), grads):
        assert (got is None) == (name not in want), name
        if got is not None:
            check(name, got, want[name], t if name in ("dpost", "dnext", "dgate") else 0)


# the types of one call that have kernels of their own: (y, residual, weights, gate), normed
FIXED = [((BF16, F32, F32, BF16), BF16), ((BF16, BF16, BF16, BF16), BF16), ((BF16, BF16, F32, BF16), BF16),
         ((F16, F16, F16, F16), F16), ((F16, F16, F32, F16), F16), ((F32, F32, F32, F32), F32)]


@pytest.mark.parametrize("gate", ["none", "channel", "token", "full"])
@pytest.mark.parametrize(("dtypes", "norm_dtype"), FIXED)
@pytest.mark.parametrize("h", [64, 520, 1000, 2048, 4096, 8192])
def test_fixed_types_over_many_rows(h, dtypes, norm_dtype, gate) -> None:
    """More rows than two per SM: each width takes another group of threads."""
    run(2 * SMS + 5, h, dtypes, gate, norm_dtype, seed=h)


@pytest.mark.parametrize(("dtypes", "norm_dtype"), FIXED)
@pytest.mark.parametrize(("t", "h"), [(1, 2048), (7, 520), (150, 7168)])
def test_fixed_types_over_few_rows(t, h, dtypes, norm_dtype) -> None:
    run(t, h, dtypes, "token", norm_dtype, seed=t)


@pytest.mark.parametrize(("dtypes", "gate"), [((F32, F32, F32, F32), "none"), ((F32, F32, F32, F32), "token"),
                                              ((BF16, BF16, F32, BF16), "full")])
@pytest.mark.parametrize("h", [4104, 7168, 8192])
def test_wide_rows_one_at_a_time(h, dtypes, gate) -> None:
    """One row per SM fits beside the weights: the same stage is filled again for each of the SM's rows."""
    run(2 * SMS + 100, h, dtypes, gate, dtypes[1], seed=h)


@pytest.mark.parametrize("dtypes", [(BF16, BF16, F32, BF16), (F32, F32, F32, F32)])
@pytest.mark.parametrize("rows", [2 * SMS, 2 * SMS + 1])
def test_either_side_of_the_change_of_forward_kernels(rows, dtypes) -> None:
    run(rows, 1024, dtypes, "channel", dtypes[1], seed=rows)
    # within one form a row is the same bits whatever the others are
    i = make(rows, 1024, dtypes, "none", seed=rows)
    x, w = i["residual"], i["next_weight"]
    more = torch.cat([x, x[:rows // 3]]) if rows > 2 * SMS else x[:rows // 2]
    n = min(len(more), rows)
    assert torch.equal(rms_norm(x, w)[:n], rms_norm(more, w)[:n])
