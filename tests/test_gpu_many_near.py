"""Attention over shared prefixes and low-rank adapters on the device, held to bounds that bf16 operands or weights and lost
tokens do not meet (test_many_near.py shows it)."""
import ctypes as C

import numpy as np
import pytest

from atlas_amd._lib import LoraC, check
from tests import many_near
from tests.gpu_util import Dev, lib
from tests.test_gpu_many import Adapters, Batch, _near

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name,window,kw", many_near.CASES, ids=[c[0] for c in many_near.CASES])
@pytest.mark.parametrize("hints", [False, True])
def test_prefix_attention_near(name, window, kw, hints):
    b = Batch(**kw).upload(hints=hints)
    out = Dev(np.full(b.q.shape, 7, np.float32))
    b.call(out, window)
    want, off = many_near.want(b, window)
    _near(out.get().reshape(want.shape), want, off)


@pytest.mark.parametrize("name,kw", many_near.LORA_CASES, ids=[c[0] for c in many_near.LORA_CASES])
def test_lora_near(name, kw):
    a = Adapters(**kw)
    d = [Dev(x) for x in (*a.raw, a.scales, a.pick, a.x, a.base)]
    y = Dev(np.full(a.base.shape, 7, np.float32))
    c = LoraC(1 if a.fmt == "bf16" else 0, d[0].ptr, d[1].ptr, d[2].ptr, a.n, a.rank, a.m, a.k)
    check(lib().atlas_lora_add_f32(C.byref(c), d[3].ptr, d[4].ptr, a.k, d[5].ptr, a.m, y.ptr, a.m, len(a.pick)))
    _near(y.get(), *many_near.lora_near(a))
