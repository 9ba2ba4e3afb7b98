"""CPU: a gradient's place that shares memory with the logits without being theirs is refused before anything is launched."""
import pytest

from wide_deep_amd import capi, policy

BASE, T, V = 1 << 30, 8, 16


def _call(name, ld, grad, ldg, size, rows=T):
    q = policy._ROWS.pack(BASE, ld, rows, V, 64, 64, 2, 0 if size == 4 else 2, 0)
    if name == "wd_pref_loss_fwd_bwd":
        o = policy._PREF.pack(0, 0, 64, 64, 64, 64, 64, grad, ldg, 0.1, 0.0, 0.0, 1.0, 1.0, 0, 0, 0)
    else:
        o = policy._POLICY.pack(64, 0, 64, 64, 64, grad, ldg, 0.2, 0.2, 0.0, 1.0, 0, 0, 0, 0)
    with pytest.raises(capi.WdError) as e:               # no device here: what is not refused fails at its launch
        capi.call(name, q, o, 64, None)
    return "shares memory" in str(e.value)


def _shares(ld, grad, ldg, size, rows):
    mine = {BASE + (r * ld + v) * size + b for r in range(rows) for v in range(V) for b in range(size)}
    return any(grad + (r * ldg + v) * size + b in mine for r in range(rows) for v in range(V) for b in (0, size - 1))


@pytest.mark.parametrize("name", ["wd_pref_loss_fwd_bwd", "wd_policy_loss_fwd_bwd"])
@pytest.mark.parametrize("size", [4, 2])
def test_overlaps(name, size):
    import torch
    if torch.cuda.is_available():
        pytest.skip("addresses are made up: only where nothing can be launched")
    for ld in (V, V + 1, 2 * V, 2 * V + 3, 5 * V):
        for ldg in (V, V + 1, 2 * V, 2 * V + 3, 5 * V):
            for off in (0, 1, V - 1, V, V + 1, 2 * V, 2 * V + 3, 3 * V, 7 * ld, 8 * ld, 7 * ld + V, -1, -V, -V + 1, -ldg, -7 * ldg, -7 * ldg - V, -8 * ldg):
                for rows in (1, 2, T):
                    grad = BASE + off * size
                    own = off == 0 and (ld == ldg or rows == 1)
                    assert _call(name, ld, grad, ldg, size, rows) == (not own and _shares(ld, grad, ldg, size, rows)), (ld, ldg, off, rows)
