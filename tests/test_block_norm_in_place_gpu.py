"""Gradients of a block norm written over the rows that they are computed from, at every way in which a row is held: by a warp, by a block in
registers, in shared memory, and read twice (above 8192 columns)."""
import numpy as np
import pytest

from language import Space

pytestmark = pytest.mark.gpu

F32, F16 = np.float32, np.float16
PLACES = [("out_grad", "normed_grad"), ("out", "branch"), ("out", "normed_grad"), ("out_grad", "branch")]


@pytest.mark.parametrize("th,ty", [(F32, F32), (F16, F16), (F32, F16)])
@pytest.mark.parametrize("width", [40, 255, 1001, 4096, 6000, 8200, 16383, 16384])
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_gradients_over_what_is_read(backend, th, ty, width, kind):
    """The bits are those of separate results, sums over rows included; the tensors that nothing lies on keep theirs."""
    rng = np.random.default_rng(width)
    rows = 9 if width > 300 else 61
    a = {"out": th, "out_grad": th, "branch": ty, "normed_grad": ty}
    a = {k: rng.standard_normal((rows, width)).astype(t) for k, t in a.items()}
    stats = np.concatenate([rng.standard_normal((rows, 1)) * 0.1 * (kind == "layer"), rng.random((rows, 1)) + 0.5] * 2, 1).astype(F32)
    w, gate = (rng.standard_normal(width).astype(F32) for _ in range(2))

    def run(residual_on, branch_on):
        space = Space(backend)
        put = space.put
        b = {k: x.copy() for k, x in a.items()}
        residual_grad = b[residual_on] if residual_on else np.full((rows, width), np.nan, th)
        branch_grad = b[branch_on] if branch_on else np.full((rows, width), np.nan, ty)
        sums = {k: np.full(width, np.nan, F32) for k in ("post_weight_grad", "gate_grad", "pre_weight_grad") + (("post_bias_grad", "pre_bias_grad") if kind == "layer" else ())}
        backend.block_norm_backward(put(b["out"]), put(b["branch"]), put(stats), out_grad=put(b["out_grad"]), normed_grad=put(b["normed_grad"]), residual_grad=put(residual_grad),
                                    branch_grad=put(branch_grad), post_weight=put(w), gate=put(gate), pre_weight=put(w), branch_scale=0.5, kind=kind,
                                    **{k: put(x) for k, x in sums.items()})
        for k, x in b.items():
            if k not in (residual_on, branch_on):
                assert np.array_equal(space.get(x)[0], a[k]), k
        return [space.get(residual_grad)[0], space.get(branch_grad)[0]] + [space.get(x)[0] for x in sums.values()]

    apart = run(None, None)
    assert all(np.isfinite(x).all() for x in apart)
    for places in PLACES:
        for x, y in zip(apart, run(*places)):
            assert np.array_equal(x, y), places


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("width", [255, 1001, 8200, 16383])
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_results_over_what_is_read(backend, dtype, width, kind):
    """Forward, both results over both inputs, straight and crossed."""
    rng = np.random.default_rng(width)
    h, y = (rng.standard_normal((7, width)).astype(dtype) for _ in range(2))
    w = rng.standard_normal(width).astype(dtype)
    got = []
    for place in ("apart", "straight", "crossed"):
        space = Space(backend)
        put = space.put
        h2, y2, stats = h.copy(), y.copy(), np.empty((7, 4), F32)
        out, normed = {"apart": (np.empty_like(h), np.empty_like(y)), "straight": (h2, y2), "crossed": (y2, h2)}[place]
        backend.block_norm(put(h2), put(y2), out=put(out), normed=put(normed), stats=put(stats), post_weight=put(w), pre_weight=put(w), kind=kind)
        got.append([space.get(x)[0] for x in (out, normed, stats)])
    for other in got[1:]:
        for x, z in zip(got[0], other):
            assert np.array_equal(x, z)
