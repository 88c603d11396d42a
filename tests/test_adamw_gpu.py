"""AdamW steps over many tensors against plain formulas in 64 bits; 8-bit states against their definition byte by byte."""
import numpy as np
import pytest

from language import EPS, Space, check
from language_steps import byte_values, decode, moments, random_bits, update
from vkml_b200 import AdamWTensor, DeviceTensor, adamw_table

pytestmark = pytest.mark.gpu

F32, F16 = np.float32, np.float16


def tensor_of(rng, shape, grad=F32, bits=32, copy=False, offset=0, decay=0.1, lr_scale=1.0):
    """A tensor's arrays in the middle of a step, `offset` elements behind an address of 256 bytes; bytes that are anything but what is no number."""
    n = int(np.prod(shape))

    def place(values, dtype):
        view = np.zeros(n + offset + 8, dtype)[offset:offset + n].reshape(shape)
        view[...] = values
        return view

    t = {"param": place(rng.standard_normal(shape), F32), "grad": place(rng.standard_normal(shape), grad), "copy": place(0, F16) if copy else None, "decay": decay,
         "lr_scale": lr_scale, "scales": None}
    if bits == 32:
        t["first"], t["second"] = place(rng.standard_normal(shape) * 0.3, F32), place(rng.random(shape) * 0.5, F32)
        return t
    words = -(-n // 4)
    for k, signed in (("first", True), ("second", False)):
        b = rng.integers(0, 127, words * 4).astype(np.uint8)
        t[k] = (b | (rng.integers(0, 2, words * 4) << 7).astype(np.uint8) if signed else b).view(np.int32).copy()
    t["scales"] = (rng.random((-(-n // 256), 2)) * 1e-3 + 1e-5).astype(F32)
    return t


def entry(space, t):
    put = space.put
    return AdamWTensor(put(t["param"]), put(t["grad"]), put(t["first"]), put(t["second"]), scales=put(t["scales"]), copy=put(t["copy"]), weight_decay=t["decay"],
                       lr_scale=t["lr_scale"])


NAMES = ("param", "first", "second", "scales", "copy")


def after(space, t):
    r = {}
    for k in NAMES:
        if t[k] is not None:
            r[k], rest = space.get(t[k])
            assert rest, k
    return r


def steps(backend, tensors, **options):
    space = Space(backend)
    backend.adamw([entry(space, t) for t in tensors], **options)
    return [after(space, t) for t in tensors]


def before(t):
    """m and v that a step starts from, flat, in 64 bits."""
    if t["scales"] is None:
        return t["first"].reshape(-1).astype(np.float64), t["second"].reshape(-1).astype(np.float64)
    n = t["param"].size
    return decode(t["first"], t["scales"][:, 0], n), decode(t["second"], t["scales"][:, 1], n) ** 2


def compare(t, got, number, lr, step, beta1=0.9, beta2=0.999, eps=1e-8, scale=1.0, seed=0):
    n = t["param"].size
    m, v = before(t)
    g = t["grad"].reshape(-1).astype(np.float64) * scale
    m, v = moments(g, m, v, beta1, beta2)
    m = (m[0], m[1] + 2 * EPS * np.abs((1 - beta1) * g) + 4 * EPS * np.abs(m[0] - (1 - beta1) * g))  # (the gradient's scale; a byte's value times its block's)
    v = (v[0], v[1] * 2)
    p, bound = update(t["param"].reshape(-1), m, v, lr * t["lr_scale"], t["decay"], step, beta1, beta2, eps)
    check(got["param"].reshape(-1), p, bound, F32, "param")
    if t["copy"] is not None:
        assert np.array_equal(got["copy"], got["param"].astype(F16))
    if t["scales"] is None:
        check(got["first"].reshape(-1), *m, F32, "first")
        check(got["second"].reshape(-1), *v, F32, "second")
        return
    # the bytes: a block's scale, and each value over it between the byte below and the one above, up by the element's bits
    bits = random_bits(seed, step, number, n)
    grid = byte_values()[:127]
    root = np.sqrt(v[0])
    root_error = v[1] / np.maximum(root, 1e-300) + 2 * EPS * root
    for k, (value, error), r in (("first", m, bits & np.uint64(0xFFFF)), ("second", (root, root_error), bits >> np.uint64(16))):
        code = got[k].view(np.uint8)[:n]
        assert np.array_equal(got[k].view(np.uint8)[n:], t[k].view(np.uint8)[n:])  # bytes behind the last element
        scales = got["scales"][:, 0 if k == "first" else 1].astype(np.float64)
        size, error = np.pad(np.abs(value), (0, -n % 256)).reshape(-1, 256), np.pad(error, (0, -n % 256)).reshape(-1, 256)
        most = size.max(1)
        assert np.all(np.abs(scales - most / 448) <= error.max(1) / 448 + 4 * EPS * most / 448), k
        zero = most < 2.0 ** -100
        inverse, error_of_most = np.where(zero, 0, 448 / np.where(zero, 1, most))[:, None], np.where(zero, 0, error.max(1) / np.where(zero, 1, most))[:, None]
        x = size * inverse
        off = (error * inverse + 8 * EPS * x + error_of_most * x).reshape(-1)[:n]
        x = x.reshape(-1)[:n]
        share = (r.astype(np.float64) * 16 + 8) / 2 ** 20

        def byte(x):
            """Up or down to the bytes' values: never falls as x rises."""
            spacing = 2.0 ** (np.floor(np.log2(np.maximum(x, 2.0 ** -6))) - 3)
            y = np.minimum(np.floor(x / spacing + share) * spacing, 448)
            return np.where((x > 0) & (y == 0), 2.0 ** -9, y) if k == "second" else y

        low, high, mine = byte(np.maximum(x - off, 0)), byte(x + off), grid[code & 127]
        if k == "second":
            low = np.where(x > 0, np.maximum(low, 2.0 ** -9), low)
        assert np.all((mine >= low) & (mine <= high)), (k, np.flatnonzero((mine < low) | (mine > high))[:5])
        # (nearly every byte is decided by this: off is 40 EPS of x or so and a byte's step 1/16 of it at least, so that 1e-4 of all values lie so near to where
        # bytes change; a few more are no surprise where there are few)
        assert np.sum(low != high) <= 4 + 1e-3 * n
        sign = code >> 7
        assert not sign.any() if k == "second" else np.array_equal(sign[np.abs(value) > m[1]], (value < 0)[np.abs(value) > m[1]])


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("grad", [F32, F16])
@pytest.mark.parametrize("copy", [False, True])
def test_a_step(backend, bits, grad, copy):
    """Sizes from one element on, more than one block's, and addresses of every alignment, in one call."""
    rng = np.random.default_rng(bits)
    shapes = [(1,), (3,), (255,), (256,), (257,), (1000,), (64, 64), (33, 77), (8192,), (4, 5, 6, 7), (100, 1001), (1 << 17,), (300, 2050)]
    tensors = [tensor_of(rng, s, grad, bits, copy, offset=o, decay=d, lr_scale=f) for s in shapes for o, d, f in ((0, 0.1, 1.0), (1, 0.0, 0.5))]
    options = dict(lr=1e-2, step=7, grad_scale=0.5, seed=99)
    for i, (t, got) in enumerate(zip(tensors, steps(backend, tensors, **options))):
        compare(t, got, i, 1e-2, 7, scale=0.5, seed=99)


@pytest.mark.parametrize("size", [1.0, 1e-4, 1e6])
def test_bytes_are_what_the_formulas_give_in_32_bits(backend, size):
    """Operation by operation in F32, each rounded by itself: the same bytes and scales, not only near ones.  (Sizes of the second form of the scaling too.)"""
    rng = np.random.default_rng(12)
    t = tensor_of(rng, (70, 1001), F32, 8)
    t["grad"] *= F32(size)
    t["scales"] *= F32(size)
    got = steps(backend, [t], lr=0.01, step=4, seed=77, grad_scale=0.75)[0]
    n, f = t["param"].size, F32
    values = byte_values().astype(f)
    of = lambda k, i: values[t[k].view(np.uint8)[:n]] * np.repeat(t["scales"][:, i], 256)[:n]  # noqa: E731
    g = t["grad"].reshape(-1) * f(0.75)
    m, r = of("first", 0), of("second", 1)
    m = m * f(0.9) + g * f(1 - 0.9)
    r = np.sqrt(r * r * f(0.999) + g * g * f(1 - 0.999))
    bits = random_bits(77, 4, 0, n).astype(np.uint32)
    for k, i, x, draw in (("first", 0, m, bits & 0xFFFF), ("second", 1, r, bits >> 16)):
        assert x.dtype == f
        most = np.pad(np.abs(x), (0, -n % 256)).reshape(-1, 256).max(1)
        assert np.array_equal(got["scales"][:, i], most * f(1 / 448))
        y = np.abs(x) * np.repeat(f(1) / most * f(448), 256)[:n]
        whole = (y * f(2.0 ** -120)).view(np.uint32)
        code = np.minimum((whole + (draw << 4 | 8)) >> 20, 126)
        if k == "second":
            code = np.where(x > 0, np.maximum(code, 1), code)
        else:
            code = np.where(np.signbit(x), code + 128, code)
        wrong = got[k].view(np.uint8)[:n] != code
        # (a value below 2^-6 of the scale's unit is rounded twice here, to a float and to a subnormal one, and once by the kernel where one product scales it)
        assert wrong.sum() <= (0 if size > 1e5 else 2), (k, wrong.sum())


@pytest.mark.parametrize("step,beta1,beta2,eps", [(1, 0.9, 0.999, 1e-8), (2, 0.0, 0.95, 1e-6), (100000, 0.9, 0.999, 1e-3), (1 << 40, 0.99, 0.0, 1e-8), (3, 0.9, 0.9999999, 1e-12)])
@pytest.mark.parametrize("bits", [32, 8])
def test_steps_and_betas(backend, step, beta1, beta2, eps, bits):
    """The first step, the last, and numbers that are given by tensors on the device."""
    rng = np.random.default_rng(3)
    tensors = [tensor_of(rng, s, F32, bits) for s in ((700,), (30, 40))]
    options = dict(beta1=beta1, beta2=beta2, eps=eps, seed=5)
    host = steps(backend, tensors, lr=0.01, step=step, grad_scale=2.0, **options)
    for i, (t, got) in enumerate(zip(tensors, host)):
        compare(t, got, i, 0.01, step, beta1, beta2, eps, 2.0, 5)
    one = lambda x, dtype: DeviceTensor.from_host(backend, np.array([x], dtype))  # noqa: E731
    device = steps(backend, tensors, lr=one(0.01, F32), step=one(step, np.int64), grad_scale=one(2.0, F32), **options)
    for i, (t, got, same) in enumerate(zip(tensors, device, host)):
        compare(t, got, i, float(F32(0.01)), step, beta1, beta2, eps, 2.0, 5)
        for k in ("first", "second", "scales"):
            assert k not in got or np.array_equal(got[k], same[k])


def test_steps_that_change_nothing(backend):
    """A scale on the device that is not finite, a step below 1 there."""
    rng = np.random.default_rng(4)
    one = lambda x, dtype: DeviceTensor.from_host(backend, np.array([x], dtype))  # noqa: E731
    for bits in (32, 8):
        t = tensor_of(rng, (50, 50), F16, bits, copy=True)
        for options in (dict(step=3, grad_scale=one(np.nan, F32)), dict(step=3, grad_scale=one(np.inf, F32)), dict(step=one(0, np.int64)), dict(step=one(-5, np.int64))):
            got = steps(backend, [t], lr=0.1, **options)[0]
            for k, x in got.items():
                assert np.array_equal(x, t[k]), (bits, k)


def test_many_tensors(backend):
    """More than a launch's parameters hold, empty ones among them."""
    rng = np.random.default_rng(5)
    tensors = [tensor_of(rng, (int(n),), F32, 8 if i % 3 else 32) for i, n in enumerate(rng.integers(0, 400, 1000))]
    for i, (t, got) in enumerate(zip(tensors, steps(backend, tensors, lr=0.01, step=2, seed=1))):
        if t["param"].size:
            compare(t, got, i, 0.01, 2, seed=1)
    backend.adamw([], lr=0.1, step=1)


def test_a_table_serves_all_steps(backend):
    rng = np.random.default_rng(6)
    tensors = [tensor_of(rng, (40, 10)), tensor_of(rng, (7,), F16, 8, True)]
    spaces = Space(backend), Space(backend)
    table = adamw_table([entry(spaces[0], t) for t in tensors])
    for step in range(1, 4):
        backend.adamw(table, lr=0.01, step=step, seed=3)
        backend.adamw([entry(spaces[1], t) for t in tensors], lr=0.01, step=step, seed=3)
    for t in tensors:
        for (k, a), b in zip(after(spaces[0], t).items(), after(spaces[1], t).values()):
            assert np.array_equal(a, b), k


@pytest.mark.parametrize("shape", [(512,), (37, 11)])
def test_values_that_are_no_numbers(backend, shape):
    """In F32 they stay with their element, in 8 bits with their block."""
    rng = np.random.default_rng(7)
    for value in (np.nan, np.inf, -np.inf):
        t, same = tensor_of(rng, shape), tensor_of(rng, shape, bits=8)
        for x in (t, same):
            x["grad"].reshape(-1)[5] = value
        got, eight = steps(backend, [t, same], lr=0.01, step=1)
        for k in ("param", "first", "second"):
            bad = ~np.isfinite(got[k].reshape(-1))
            assert bad[5] and bad.sum() == 1, k
        n = t["param"].size
        for k, i in (("first", 0), ("second", 1)):
            assert np.isnan(eight["scales"][0, i]) and np.isfinite(eight["scales"][1:, i]).all()
            codes = eight[k].view(np.uint8)[:n] & 127
            assert np.all(codes[:min(n, 256)] == 127) and not np.any(codes[256:] == 127)
        assert np.isfinite(np.delete(eight["param"].reshape(-1), 5)).all()


def test_blocks_of_zeros_and_of_tiny_values(backend):
    rng = np.random.default_rng(8)
    for size in (0.0, 1e-45, 2.0 ** -101, 1e-25, 1e15):
        t = tensor_of(rng, (600,), F32, 8)
        t["first"][...], t["second"][...], t["scales"][...] = 0, 0, 0
        t["grad"][...] = rng.standard_normal(600) * size
        got = steps(backend, [t], lr=0.01, step=1, beta1=0.5, beta2=0.5, eps=1e-20)[0]
        if size < 2.0 ** -99:
            assert not got["scales"].any() or size == 2.0 ** -101
        if 1e-20 < size or size == 0.0:
            compare(t, got, 0, 0.01, 1, 0.5, 0.5, 1e-20)
        assert np.isfinite(got["param"]).all()


def test_small_changes_are_kept_on_average(backend):
    """A change of a small part of a byte's step moves as many bytes as it is a part of a step: 4 standard deviations of such a count, and 16 bits' own step."""
    n = 1 << 17
    rng = np.random.default_rng(9)
    for code, g in ((0x60, 6e-3), (0x60, 2e-3), (0x31, 3e-4), (0x05, 1e-5)):
        t = tensor_of(rng, (n,), F32, 8)
        t["scales"][...], t["grad"][...] = 2e-5, g
        c = np.full(n, code, np.uint8)
        c[::256] = 0x7E  # one large value keeps each block's scale
        t["first"], t["second"] = np.zeros(n // 4, np.int32), c.view(np.int32).copy()
        t["grad"][::256] = 448 * 2e-5
        got = steps(backend, [t], lr=0.0, step=1, seed=4)[0]
        grid, scale = byte_values(), float(F32(2e-5))
        r = np.sqrt(0.999 * (grid[code] * scale) ** 2 + 0.001 * float(F32(g)) ** 2) / scale
        low = np.searchsorted(grid[:127], r, side="right") - 1
        part = (r - grid[low]) / (grid[low + 1] - grid[low])
        others = got["second"].view(np.uint8)[np.arange(n) % 256 != 0]
        assert set(np.unique(others)) <= {low, low + 1}
        count = len(others)
        assert abs(np.mean(others == low + 1) - part) <= 4 * np.sqrt(part * (1 - part) / count) + 2.0 ** -16 + 1e-5, (code, g, part)


def test_the_same_bits_again_and_others_of_another_seed(backend):
    rng = np.random.default_rng(10)
    t = tensor_of(rng, (300, 70), F16, 8, True)
    a, b, c, d = (steps(backend, [t], lr=0.01, step=s, seed=k)[0] for s, k in ((5, 1), (5, 1), (5, 2), (6, 1)))
    assert all(np.array_equal(a[k], b[k]) for k in a)
    for other in (c, d):
        assert np.mean(a["first"].view(np.uint8) != other["first"].view(np.uint8)) > 0.2


def test_a_tensor_beyond_32_bits(backend):
    """More than 2^31 elements in one tensor, 8-bit states: the blocks at its end."""
    n = (1 << 31) + 1000 - 1000 % 256
    sizes = {"param": 4 * n, "grad": 2 * n, "first": -(-n // 4) * 4, "second": -(-n // 4) * 4, "scales": -(-n // 256) * 8}
    from vkml_b200 import DType, TensorDesc
    storage = {k: backend.allocate(s) for k, s in sizes.items()}
    tail, at = 256 * 7, n - 256 * 7
    rng = np.random.default_rng(11)
    t = tensor_of(rng, (tail,), F16, 8)
    backend.copy_from_host(storage["param"], 4 * at, t["param"])
    backend.copy_from_host(storage["grad"], 2 * at, t["grad"])
    backend.copy_from_host(storage["first"], at, t["first"])
    backend.copy_from_host(storage["second"], at, t["second"])
    backend.copy_from_host(storage["scales"], at // 256 * 8, t["scales"])
    desc = lambda k, dims, dtype: TensorDesc.contiguous(storage[k].data, dims, dtype)  # noqa: E731
    backend.adamw([AdamWTensor(desc("param", (n,), DType.F32), desc("grad", (n,), DType.F16), desc("first", (-(-n // 4),), DType.I32), desc("second", (-(-n // 4),), DType.I32),
                               scales=desc("scales", (-(-n // 256), 2), DType.F32), weight_decay=0.1)], lr=0.01, step=3, seed=2)
    got = np.zeros(tail, F32)
    backend.copy_to_host(got, storage["param"], 4 * at)
    m, v = before(t)
    m, v = moments(t["grad"].astype(np.float64), m, v, 0.9, 0.999)
    p, bound = update(t["param"], (m[0], m[1] + 8 * EPS * np.abs(m[0]) + 8 * EPS * np.abs(t["grad"])), (v[0], v[1] * 2), 0.01, 0.1, 3, 0.9, 0.999, 1e-8)
    check(got, p, bound, F32, "param")
    code = np.zeros(tail, np.uint8)
    backend.copy_to_host(code, storage["first"], at)
    scales = np.zeros((7, 2), F32)
    backend.copy_to_host(scales, storage["scales"], at // 256 * 8)
    new = byte_values()[code] * np.repeat(scales[:, 0].astype(np.float64), 256)[:tail]
    assert np.abs(new - m[0]).max() <= np.repeat(scales[:, 0], 256).max() * 32
