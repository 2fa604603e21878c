"""The bound of the 4-bit attention's accuracy: parts that are lost pass it (planted in the NumPy form, without a device)."""
import pytest

from tests import kv4_parts
from tests.test_gpu_kv4 import Case


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("form", kv4_parts.FORMS)
def test_lost_parts_pass_the_bound(hd, form):
    c, heads, q = kv4_parts.case(Case, hd, form)
    n, every = kv4_parts.q_parts(hd), {"prompt16": 3, "prompt32": 11, "runs32": 5}.get(form, 1)

    def parts(n_q, n_p):
        _, want, size, got = kv4_parts.outputs(c, heads, q, hd ** -0.5, n_q, n_p, every)
        return got, want, size

    limit = kv4_parts.limit(*parts(n, 3))
    assert kv4_parts.error(*parts(n, 3)) < limit / 4
    assert kv4_parts.error(*parts(n - 2, 3)) > limit and kv4_parts.error(*parts(n, 2)) > limit
