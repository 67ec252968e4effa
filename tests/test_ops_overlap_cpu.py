"""constrain_logits takes out in the logits' own place or apart from them;
anything between is refused before a device is touched (no GPU needed)."""
import pytest

import gateddeltanet_b200 as gdn
from test_ops_cpu import FAKE, lib, logits_args  # noqa: F401


@pytest.mark.parametrize("change", [
    dict(out=FAKE + 4), dict(out=FAKE - 4), dict(out=FAKE + 400), dict(out=FAKE, out_row=101), dict(out=FAKE + 99 * 4, rows=1),
    dict(out=FAKE - 2 * 99, dtype=1), dict(logits_row=220, out_row=220, out=FAKE + 4 * 99),
    dict(logits_row=220, out_row=220, out=FAKE + 4 * 121), dict(logits_row=0, out=FAKE + 4 * 50),
    dict(logits_row=220, out_row=300, out=FAKE + 4 * 110)], ids=str)
def test_partly_shared_memory_is_refused(lib, change):  # noqa: F811
    assert lib.gdn_b200_constrain_logits(logits_args(**change)) == -1
    assert "overlaps" in gdn.last_error()


@pytest.mark.parametrize("change", [
    dict(), dict(out=FAKE + 800), dict(out=FAKE - 800), dict(out=FAKE + 400, rows=1), dict(logits_row=220, out_row=220, out=FAKE + 4 * 100),
    dict(logits_row=220, out_row=220, out=FAKE - 4 * 100), dict(logits_row=220, out_row=220, out=FAKE + 4 * 120),
    dict(logits_row=0, out=FAKE + 400)], ids=str)
def test_the_same_place_or_another_is_taken(lib, change):  # noqa: F811
    assert lib.gdn_b200_constrain_logits(logits_args(**change, device=77)) == -1
    assert "device" in gdn.last_error()  # refused for the device alone
