"""Every form of the row attention's kernels (row_forms.py) against the plain 64-bit form: trees and causal chunks,
one row with weights, each kind of score rule. Of many streams only three have rows: the others' are left as they were."""

import ctypes as C

import numpy as np
import pytest

from tests import attention_ref as ref
from tests import row_forms as forms
from tests.test_gpu_tree_cache import RULE, TABLE, Gpu, caches, masks

pytestmark = pytest.mark.gpu


@pytest.fixture()
def gpu():
    g = Gpu()
    yield g
    g.free()


def streams_of(gpu, b, live, x):
    """A device array of b streams whose `live` ones hold x."""
    L, p, size = gpu.hip.lib(), C.c_void_p(), x[0].nbytes
    gpu.hip._check(L.hs_device_alloc(gpu.dev.h, b * size, C.byref(p)))
    gpu.held.append(p)
    for i, s in enumerate(live):
        gpu.hip._check(L.hs_device_upload(gpu.dev.h, C.c_void_p(p.value + s * size), gpu.hip._ptr(np.ascontiguousarray(x[i])), size))
    return p


def run(gpu, b, t, h, hd, cap, score_s, tree):
    kind = forms.form(b, t, h, hd, cap, score_s, not tree)
    print(f"{'tree' if tree else 'mass'} {b}x{t}x{h}x{hd} cap {cap} shift {score_s}: {kind}", flush=True)
    r = np.random.default_rng(b + t + hd + cap + score_s)
    rule = (forms.SCORES[score_s], score_s, *RULE[2:])
    live = [0, b // 2, b - 1]
    n = len(live)
    q = r.integers(-128, 128, (n, t, h, hd)).astype(np.int8)
    kc, vc = caches(r, n, h, cap, hd)
    rows = np.array([t, max(1, t // 2), max(1, t - 1)], np.uint32)
    ctx = np.array([cap - t, cap // 3, 65], np.uint32) + (0 if tree else rows)
    ctx = np.minimum(ctx, cap).astype(np.uint32)

    def spread(x, fill=0):
        out = np.full((b, *x.shape[1:]), fill, x.dtype)
        out[live] = x
        return out

    out = np.full((n, t, h, hd), 77, np.int8)
    all_out = spread(out, 77)
    d = [gpu(spread(q)), streams_of(gpu, b, live, kc), streams_of(gpu, b, live, vc), gpu(spread(ctx)), gpu(spread(rows))]
    d_out, g_rule, dims = gpu(all_out), gpu.rule(rule, TABLE), (b, t, h, hd, cap)
    if tree:
        mask = masks(gpu, r, n, t, empty=0.05)
        gpu.hip.attend_tree(gpu.dev, *d, gpu(spread(mask)), dims, g_rule, d_out)
        ref.tree(q, kc, vc, ctx, rows, mask, rule, TABLE, out)
    else:
        acc = r.integers(0, 2 ** 40, (n, h, cap)).astype(np.uint64)
        d_acc = gpu(spread(acc))
        gpu.hip.attend_mass(gpu.dev, *d, d_acc, dims, g_rule, d_out)
        ref.mass(q, kc, vc, ctx, rows, acc, rule, TABLE, out)
        everyone = np.zeros((b, h, cap), np.uint64)
        assert np.array_equal(gpu.back(d_acc, everyone), spread(acc))
    assert np.array_equal(gpu.back(d_out, all_out), spread(out, 77))


@pytest.mark.parametrize("score_s", sorted(forms.SCORES))
@pytest.mark.parametrize("shape", forms.SHAPES)
def test_rows(gpu, shape, score_s):
    run(gpu, *shape, score_s, True)
    run(gpu, *shape, score_s, False)


@pytest.mark.parametrize("score_s", sorted(forms.SCORES))
@pytest.mark.parametrize("b,h,hd,cap", forms.ONE_ROW)
def test_one_row(gpu, b, h, hd, cap, score_s):
    run(gpu, b, 1, h, hd, cap, score_s, False)
