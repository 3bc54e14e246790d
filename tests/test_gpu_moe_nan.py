"""A token whose router logits are not numbers, among others: it is flagged, and the others' rows are what they are without it."""
import numpy as np
import pytest

import eahmmf_b200 as eb
import synth

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("E,K", [(16, 4), (128, 8)])
@pytest.mark.parametrize("T", [1, 2, 3, 4, 8, 20, 64, 100])
@pytest.mark.parametrize("fill", ["all", "one", "infinities"])
def test_nan_logits_are_flagged_and_alone(E, K, T, fill):
    import torch
    if not torch.cuda.is_available():
        pytest.fail("CUDA device required")
    ex = synth.expert_set(D=512, FF=256, n_expert=E, seed=42)
    layer = eb.MoeLayer.from_expert_set(ex, n_used=K)
    x, xn, lg = synth.activations(T, 512, seed=1), synth.activations(T, 512, seed=2), synth.router_logits(T, E, seed=3)

    def run(logits):
        dx = torch.from_numpy(x.copy()).cuda()
        ws = torch.zeros(layer.workspace_bytes(T), dtype=torch.uint8, device="cuda")
        st = torch.zeros(1, dtype=torch.int32, device="cuda")
        assert layer(T, torch.from_numpy(xn).cuda(), torch.from_numpy(logits).cuda(), dx, ws, d_status=st) == 0
        torch.cuda.synchronize()
        return dx.cpu().numpy(), int(st.item())

    want, st = run(lg)
    assert st == 0
    bad = lg.copy()
    rows = [T // 2] if T < 20 else [0, T // 2, T - 1]
    for t in rows:
        if fill == "all":
            bad[t] = np.nan
        elif fill == "one":
            bad[t, E // 3] = np.nan
        else:
            bad[t, [1, 5]] = np.inf
    got, st = run(bad)
    assert st == eb.ST_BAD_INDEX
    keep = [t for t in range(T) if t not in rows]
    np.testing.assert_array_equal(got[keep], want[keep])
