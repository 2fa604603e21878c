"""The bound of the 4-bit attention's accuracy: parts that are lost pass it (planted in the NumPy form, without a device)."""
import pytest

from tests import kv4_parts
from tests.test_gpu_kv4 import Case


def _parts(c, heads, q, scale, every, n_q, n_p):
    _, want, size, got = kv4_parts.outputs(c, heads, q, scale, n_q, n_p, every)
    return got, want, size


def _every(form):
    return {"prompt16": 3, "prompt32": 11, "runs32": 5}.get(form, 1)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("form", kv4_parts.FORMS)
def test_lost_parts_pass_the_bound(hd, form):
    args = kv4_parts.case(Case, hd, form) + (hd ** -0.5, _every(form))
    n = kv4_parts.Q_PARTS
    limit = kv4_parts.limit(*_parts(*args, n, 3))
    assert kv4_parts.error(*_parts(*args, n, 3)) < limit / 4
    assert kv4_parts.error(*_parts(*args, n - 2, 3)) > limit and kv4_parts.error(*_parts(*args, n, 2)) > limit


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("form", kv4_parts.SHORT_FORMS)
def test_one_lost_part_of_q_passes_the_bound(hd, form):
    args = kv4_parts.short_case(Case, hd, form) + (kv4_parts.SHORT_SCALE * hd ** -0.5, 1)
    n = kv4_parts.Q_PARTS
    limit = kv4_parts.limit(*_parts(*args, n, 3), kv4_parts.SHORT_STEPS, 2)
    assert kv4_parts.error(*_parts(*args, n, 3)) < limit / 2 and kv4_parts.error(*_parts(*args, n - 1, 3)) > limit
