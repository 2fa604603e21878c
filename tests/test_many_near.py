"""The bounds of many_near on the CPU: 32 bits are within them, and operands or weights of fewer bits and
lost tokens are not."""
import numpy as np
import pytest

from tests import many_near
from tests.test_gpu_many import Adapters, Batch


def _in_32_bits(b, window=0, drop=(), weights=np.float32):
    """Each row's attention as numpy's float32 makes it, without the tokens at the positions of drop."""
    q = b.q.reshape(-1, b.n_kv, b.heads // b.n_kv, b.hd) * np.float32(b.hd ** -0.5)
    got = np.zeros((len(q), b.heads, b.hd), np.float32)
    for g in range(len(b.prefix)):
        for r in range(b.starts[g], b.starts[g + 1]):
            t = np.setdiff1d(np.arange(max(0, b.lens[r] - window) if window else 0, b.lens[r]), drop)
            i = t - b.prefix[g]
            at = np.where(i < 0, b.prefix_slots[g], b.slots[r, np.maximum(i, 0)]), t
            k, v = (x[at].transpose(1, 0, 2) for x in (b.k, b.v))
            s = q[r] @ k.transpose(0, 2, 1)
            p = np.exp(s - s.max(-1, keepdims=True))
            p = many_near.bf16(p) if weights == "bf16" else p
            got[r] = ((p @ v) / p.sum(-1, keepdims=True)).reshape(b.heads, b.hd)
    return got


def _off(b, got, window):
    want, off = many_near.want(b, window)
    return (np.abs(got - want) / off).max()


@pytest.fixture(scope="module", params=many_near.CASES, ids=lambda c: c[0])
def case(request):
    _, window, kw = request.param
    return Batch(junk=False, **kw), window


def test_32_bits_are_near(case):
    b, window = case
    assert _off(b, _in_32_bits(b, window), window) < 0.1


@pytest.mark.parametrize("what", ["k", "v", "q"])
def test_operands_in_bf16_are_not(case, what):
    b, window = case
    want, off = many_near.want(b, window)
    full = getattr(b, what)
    try:
        setattr(b, what, many_near.bf16(full))
        got = _in_32_bits(b, window)
    finally:
        setattr(b, what, full)
    assert (np.abs(got - want) / off).max() > 2


def test_weights_in_bf16_are_not(case):
    b, window = case
    assert _off(b, _in_32_bits(b, window, weights="bf16"), window) > 2


@pytest.mark.parametrize("where", ["first", "middle", "last shared", "first own"])
def test_a_lost_token_is_not(case, where):
    b, window = case
    n, first = int(b.prefix[0]), max(0, int(b.lens.max()) - window) if window else 0
    at = {"first": first, "middle": (first + n) // 2, "last shared": n - 1, "first own": n}[where]
    assert _off(b, _in_32_bits(b, window, [at]), window) > 2


@pytest.fixture(params=many_near.LORA_CASES, ids=lambda c: c[0])
def adapters(request):
    return Adapters(**request.param[1])


def _lora_in_32_bits(a, x, low=lambda v: v):
    y = a.base.copy()
    for r, p in enumerate(a.pick):
        if 0 <= p < a.n:
            y[r] += a.scales[p] * (a.b[p] @ low(a.a[p] @ x[r]))
    return y


def test_adapters_in_32_bits_are_near_and_in_bf16_are_not(adapters):
    a = adapters
    want, off = many_near.lora_near(a)
    assert (np.abs(_lora_in_32_bits(a, a.x) - want) / off).max() < 0.5
    assert (np.abs(_lora_in_32_bits(a, many_near.bf16(a.x)) - want) / off).max() > 2
    assert (np.abs(_lora_in_32_bits(a, a.x, many_near.bf16) - want) / off).max() > 2
