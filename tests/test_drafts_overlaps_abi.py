"""CPU: verify_drafts refuses a workspace that lies over its results or over anything that it reads."""
import pytest

import nedo_gpu
from test_q4_drafts_abi import drafts

WS, ROWS = 1 << 24, 6  # an aligned, never read address


def refused(lib, temperature=1.0, accepted=1 << 20, ids=1 << 21, **kw):
    d = drafts(rows=ROWS, **kw)
    with pytest.raises(nedo_gpu.NedoGpuError, match="the workspace overlaps") as e:
        lib.verify_drafts_dev(d, temperature, accepted, ids, WS, lib.verify_drafts_workspace(d))
    assert e.value.code == nedo_gpu.ERR_ARG


@pytest.mark.parametrize("temperature", [0.0, 1.0])
def test_workspace_over_results_refused(lib, temperature):
    need = lib.verify_drafts_workspace(drafts(rows=ROWS))
    for at in (WS, WS + need - 4, WS - 4):
        refused(lib, temperature, accepted=at)
        refused(lib, temperature, ids=at)


@pytest.mark.parametrize("name,size", [("row_start", 12), ("logits", ROWS * 4000), ("draft_ids", ROWS * 4), ("draft_probs", ROWS * 4000),
                                       ("accept_u", ROWS * 4), ("sample_u", 8)])
def test_workspace_over_inputs_refused(lib, name, size):
    """Up to the last elements; at temperature 0 what that reads."""
    need = lib.verify_drafts_workspace(drafts(rows=ROWS))
    step = 16 if size > 1000 else 4
    for at in (WS, WS + need - step, WS - size + step):
        refused(lib, 1.0, **{name: at})
        if name in ("row_start", "logits", "draft_ids"):
            refused(lib, 0.0, **{name: at})
