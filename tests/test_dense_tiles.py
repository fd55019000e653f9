"""The linear layer and the gated block on every tile that their products are cut into, the largest above all.

Which tile a product gets is decided on the host, from sizes (mdn_op_dense_tiles).  TILES says what each shape here
gets; a change of the estimates behind that choice shows in a test that needs no GPU, so that no tile loses its tests
unseen.  Tolerances are those of test_dense.py, whose formulas and inputs these are."""
import ctypes
import re

import pytest
import torch  # before the library: one HIP runtime in the process
from test_dense import ACTS, BF16, F32, LEAVES, SHAPES, call, check, inputs

gpu = pytest.mark.gpu
FORWARD, SLOPES, D_X, D_W = range(4)


class _Tile(ctypes.Structure):
    _fields_ = [(n, ctypes.c_uint32) for n in ("rows", "step", "parts")]


def tiles(rows, width, out, dtype, gated, slope=True):
    """(rows, bytes of a step, parts) of the four products of a call with every gradient"""
    from mdnav import native, policy
    up = 4096 if gated else 0
    dense = policy._Dense.from_buffer_copy(policy._DENSE.pack(
        rows, width, out, int(dtype == BF16), policy.ACTIVATIONS["silu" if slope else "none"], gated, 4096, width, 4096, width, up, width,
        0, 0, 4096, out, 0, 0))
    grad = policy._DenseGrad.from_buffer_copy(policy._DENSE_GRAD.pack(4096, out, 4096, width, 4096, width, up, width, 0, 0))
    made = (_Tile * 4)()
    native.check(native.lib().mdn_op_dense_tiles(ctypes.byref(dense), ctypes.byref(grad), made))
    return [(t.rows, t.step, t.parts) for t in made]


# (rows, in, out), type, gated: the products that it is here for, and the rows of their tiles.  Rows, columns and sums
# that end inside a tile, a word and a step, and ones that do not; sums of two matrices; rows of no whole words.
TILES = [
    ((51617, 513, 157), BF16, False, {FORWARD: 256, SLOPES: 256}),
    ((52000, 640, 144), BF16, False, {FORWARD: 256, SLOPES: 256}),
    ((56827, 133, 260), BF16, False, {D_X: 256}),
    ((4318, 11029, 137), BF16, False, {D_W: 256}),
    ((287, 20270, 521), BF16, False, {D_W: 256}),
    ((49596, 304, 66), BF16, True, {FORWARD: 256, SLOPES: 256}),
    ((50000, 320, 128), BF16, True, {FORWARD: 256, SLOPES: 256}),
    ((139, 304, 26135), BF16, True, {FORWARD: 256, SLOPES: 256, D_W: 128}),
    ((52009, 135, 134), BF16, True, {D_X: 256}),
    ((14374, 203, 3935), BF16, True, {FORWARD: 256, SLOPES: 256, D_W: 256}),
    ((273, 24916, 137), BF16, True, {D_W: 256}),
    ((4205, 5847, 133), BF16, True, {D_W: 256}),
    ((23031, 33, 65), F32, False, {FORWARD: 128, SLOPES: 128}),
    ((18092, 67, 42), F32, False, {D_X: 128}),
    ((133, 11081, 151), F32, False, {D_W: 128}),
]
IDS = ["%dx%dx%d-%s%s" % (*shape, "bf16" if dtype == BF16 else "f32", "-gated" * gated) for shape, dtype, gated, _ in TILES]


@pytest.mark.parametrize("case", TILES, ids=IDS)
def test_the_tiles_of_a_shape(case):
    shape, dtype, gated, want = case
    made = tiles(*shape, dtype, gated)
    assert {i: made[i][0] for i in want} == want
    if D_W in want:  # sums in one piece and in several
        assert (made[D_W][2] > 1) == (shape[0] > 1000)


def test_what_the_choice_says():
    assert tiles(0, 64, 64, BF16, True) == 4 * [(0, 0, 0)]
    few = tiles(16, 64, 64, BF16, False, slope=False)  # the kernel of few rows, and no argument to make again
    assert few[:2] == 2 * [(0, 0, 0)] and all(t[0] == 64 and t[1] == 128 and t[2] == 1 for t in few[2:])
    assert tiles(262144, 256, 1024, BF16, True)[FORWARD] == (128, 64, 1)
    from mdnav import native
    made = (_Tile * 4)()
    assert native.lib().mdn_op_dense_tiles(None, None, made) == -1 and b"null" in native.lib().mdn_last_error()


@gpu
@pytest.mark.parametrize("case", TILES, ids=IDS)
def test_matches_the_formula(case):
    shape, dtype, gated, _ = case
    act = list(ACTS)[1 + sum(shape) % 6]
    for plain in (False, True):
        if plain and gated:
            continue
        print("case: tiles", shape, dtype, gated, "none" if plain else act, flush=True)
        check(inputs(*shape, dtype, gated, bias=True, residual=not gated and not plain, seed=sum(shape) + plain), "none" if plain else act, dtype)


def run(v, leaves, act="silu"):
    t = {n: x.detach().requires_grad_() if n in leaves else x for n, x in v.items()}
    y = call(t, act)
    return [y.detach()] + list(torch.autograd.grad(y, [t[n] for n in leaves], v["d_y"]))


@gpu
@pytest.mark.parametrize("shape,gated", [((51617, 513, 157), False), ((52000, 640, 144), False), ((14374, 203, 3935), True),
                                         ((52009, 135, 134), True), ((4318, 11029, 137), False)], ids=str)
def test_rows_apart(shape, gated):
    """Operands, residual and the result's gradient at any element of memory: the bits of contiguous ones."""
    print("case: rows apart", shape, flush=True)
    v = inputs(*shape, BF16, gated, residual=not gated, seed=21)
    leaves = [n for n in LEAVES if v[n] is not None]
    want = run(v, leaves)

    def spread(t, gap, start):
        if t is None or t.dim() < 2:
            return t
        wide = torch.full((t.shape[0], t.shape[1] + gap + start), float("nan"), dtype=t.dtype, device="cuda")
        wide[:, start:start + t.shape[1]] = t
        return wide[:, start:start + t.shape[1]]

    for gap, start in ((8, 0), (6, 1)):
        for a, b in zip(run({n: spread(t, gap, start) for n, t in v.items()}, leaves), want):
            assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("shape,gated", [((14374, 203, 3935), True), ((52009, 135, 134), True), ((49596, 304, 66), True),
                                         ((51617, 513, 157), False), ((287, 20270, 521), False)], ids=str)
def test_alone_and_again(shape, gated):
    """The same bits in every call, between others, and of each gradient by itself."""
    print("case: again", shape, flush=True)
    v, other = (inputs(*shape, BF16, gated, residual=not gated, seed=s) for s in (22, 23))
    leaves = [n for n in LEAVES if v[n] is not None]
    want = run(v, leaves)
    for _ in range(3):
        run(other, leaves)
        for a, b in zip(run(v, leaves), want):
            assert torch.equal(a, b)
    for i, n in enumerate(leaves):
        assert torch.equal(run(v, [n])[1], want[1 + i]), n


@gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("shape", [(14374, 203, 3935), (52009, 135, 134)], ids=str)
def test_bad_rows_stay_alone(shape, bad):
    v = inputs(*shape, BF16, True, seed=24)
    at = shape[0] - 3
    worse = dict(v, x=v["x"].clone())
    worse["x"][at, shape[1] - 1] = bad
    keep = torch.arange(shape[0], device="cuda") != at
    for a, b in zip(run(v, ["x"]), run(worse, ["x"])):
        assert torch.equal(a[keep], b[keep]) and not torch.isfinite(b[at]).all()


@gpu
@pytest.mark.parametrize("shape,gated", [((14374, 203, 3935), True), ((52009, 135, 134), True), ((51617, 513, 157), False)], ids=str)
def test_only_the_results_are_written(shape, gated):
    """Results with rows apart, through the C entries: what lies between and around stays."""
    from mdnav import native, policy
    print("case: written", shape, flush=True)
    L, (rows, width, out) = native.lib(), shape
    v = inputs(*shape, BF16, gated, residual=not gated, seed=25)
    leaves = [n for n in LEAVES if v[n] is not None]
    want = dict(zip(["y"] + leaves, run(v, leaves)))

    def room(n, w):  # rows an odd number of elements apart, one row before and one behind
        return torch.full((n + 2, w + 3), 7.0, dtype=BF16, device="cuda")

    made = dict(y=room(rows, out), x=room(rows, width), w=room(out, width), w_up=room(out, width) if gated else None, b=room(1, out),
                b_up=room(1, out) if gated else None)

    def at(t):
        return (0, 0) if t is None else (t[1].data_ptr(), t.shape[1])

    def given(t):
        return (0, 0) if t is None else (t.data_ptr(), t.shape[-1])

    c = policy._Dense.from_buffer_copy(policy._DENSE.pack(
        rows, width, out, 1, policy.ACTIVATIONS["silu"], gated, *given(v["x"]), *given(v["w"]), *given(v["w_up"]), *given(v["residual"]),
        *at(made["y"]), given(v["b"])[0], given(v["b_up"])[0]))
    d = policy._DenseGrad.from_buffer_copy(policy._DENSE_GRAD.pack(
        *given(v["d_y"]), *at(made["x"]), *at(made["w"]), *at(made["w_up"]), at(made["b"])[0], at(made["b_up"])[0]))
    stream = torch.cuda.current_stream().cuda_stream
    size = ctypes.c_uint64()

    def work():  # as large as asked for, something of the caller's behind it
        t = torch.full((size.value + 256,), 9, dtype=torch.uint8, device="cuda")
        return t, (t.data_ptr(), size.value)

    native.check(L.mdn_op_dense_forward_bytes(ctypes.byref(c), ctypes.byref(size)))
    first, args = work()
    native.check(L.mdn_op_dense_forward(ctypes.byref(c), *args, stream))
    assert (first[size.value:] == 9).all()
    native.check(L.mdn_op_dense_backward_bytes(ctypes.byref(c), ctypes.byref(d), ctypes.byref(size)))
    second, args = work()
    native.check(L.mdn_op_dense_backward(ctypes.byref(c), ctypes.byref(d), *args, stream))
    assert (second[size.value:] == 9).all()
    for n, t in made.items():
        if t is None:
            continue
        inner = want[n].reshape(t.shape[0] - 2, -1)
        assert torch.equal(t[1:-1, :-3], inner), n
        assert (t[0] == 7).all() and (t[-1] == 7).all() and (t[:, -3:] == 7).all(), n


@gpu
def test_captured():
    """A graph of both passes, replayed between eager calls and on changed inputs."""
    v = inputs(14374, 203, 3935, BF16, True, seed=26)
    leaves = [n for n in LEAVES if v[n] is not None]
    gen = torch.Generator(device="cuda").manual_seed(3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(v, leaves)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run(v, leaves)
    for _ in range(3):
        for n in leaves:
            v[n].copy_(torch.randn(v[n].shape, generator=gen, device="cuda") * 0.2)
        want = [t.clone() for t in run(v, leaves)]
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, want):
            assert torch.equal(a, b)


def test_every_kernel_is_reached():
    """The product kernels in the library are those that the calls of this file and of test_dense.py launch: none is
    built that no call reaches, and none is untested."""
    from mdnav import native
    LINEAR, GATED, SLOPE, GATED_SLOPE, STORE, PART = range(6)
    calls = [(shape, dtype, gated, slope) for shape, dtype, gated, _ in TILES for slope in ([True] if gated else [True, False])]
    for shape in SHAPES:
        for dtype in (F32, BF16):
            for i, gated in enumerate((False, True, False)):  # the activations that test_dense.py gives them
                calls.append((shape, dtype, gated, gated or (i != 2 and list(ACTS)[(sum(shape) + 3 * i) % len(ACTS)] != "none")))
    reached = set()
    for shape, dtype, gated, slope in calls:
        for i, (rows, step, parts) in enumerate(tiles(*shape, dtype, gated, slope)):
            if rows:
                result = [GATED if gated else LINEAR, GATED_SLOPE if gated else SLOPE, STORE, PART if parts > 1 else STORE][i]
                reached.add((dtype, rows, step, i == D_W, i >= D_X, result))
    with open(native.LIB_PATH, "rb") as f:
        names = re.findall(rb"14product_kernelI(f|DF16b)Li(\d+)ELi\d+ELi\d+ELi\d+ELi(\d+)ELi\d+ELb[01]ELb([01])ELb([01])ELi(\d)E", f.read())
    built = {(F32 if t == b"f" else BF16, int(rows), int(step), m == b"1", n == b"1", int(result)) for t, rows, step, m, n, result in names}
    assert len(built) > 30 and built == reached, (built - reached, reached - built)
