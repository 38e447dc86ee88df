import pytest

# Tests that hold a value their operator no longer gives, with the reason. They run, unchanged, and have to fail (what else they check is in the test that is named).
OUTDATED = {
    "tests/test_gpu_verify_draft.py::test_temperatures":
        "takes a drafter's row at a temperature of 1 where draft_temp <= 0. A drafter that took its greatest token has q = 1 there: accepted with u q' < p for another q' and redrawn from "
        "max(p - q', 0), what comes out does not have the target's distribution (q' = 1/2, p = 1/4 at that token: it comes out half of the time). "
        "test_gpu_verify_greedy_drafter.py::test_other_temperatures has its other calls",
}


def pytest_collection_modifyitems(items):
    for item in items:
        if item.nodeid in OUTDATED:
            item.add_marker(pytest.mark.xfail(strict=True, reason=OUTDATED[item.nodeid]))
