"""The cache's, the attention's and the drafts' functions without a GPU: arguments at the ends of what they take."""
import math

import pytest

torch = pytest.importorskip("torch")
from verinf_amd.prover import generation as gen  # noqa: E402


@pytest.mark.parametrize("bad", [dict(base=1e10, scaling=("base", 1e200)), dict(base=1e300, scaling=("base", 1e10)), dict(scaling=("linear",)), dict(scaling=2.0),
                                 dict(scaling=("parts", 2.0, 4096, math.nan, 32.0))])
def test_plans_that_have_no_frequencies(bad):
    with pytest.raises(RuntimeError, match="rotary_plan"):
        gen.rotary_plan(4, device="cpu", **bad)
