"""The tests of paged attention in test_gpu_paged_shared once more, with bounds under
which a NaN on one side alone is a difference (``paged_strict_check``)."""

import paged_scores_reference
import paged_strict_check
import pytest
from test_gpu_paged_shared import *  # noqa: F401,F403

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def strict(monkeypatch):
    monkeypatch.setattr(paged_scores_reference, "check", paged_strict_check.check)
