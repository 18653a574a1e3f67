"""The context's two streams and what is recorded on them.  Needs a real MI355X (-m gpu)."""
import pytest

from gpu_helpers import *  # noqa: F401,F403

pytestmark = pytest.mark.gpu


def test_both_streams_have_the_default_priority():
    assert pa.context().stream_priorities() == {"compute": 0, "comm": 0, "least": 0, "greatest": 0}
