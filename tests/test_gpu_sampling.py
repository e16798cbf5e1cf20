"""Sampling on the GPU against its definition in 64 bits: the same tokens, ties and
cuts included, and the same tokens as the host sampler's for its own draws."""
import math

import numpy as np
import pytest
import torch

from evo_hip import native as N

pytestmark = pytest.mark.gpu
DEVICE = "cuda:0"
CODES = {torch.float32: N.DTYPE_F32, torch.bfloat16: N.DTYPE_BF16, torch.float16: N.DTYPE_F16}
NONE = -1  # UINT32_MAX as int32


def sample(logits, uniform, temperature=None, top_k=None, top_p=None, min_p=None,
           workspace=True):
    rows, vocab = logits.shape
    ptr = lambda x: None if x is None else x.data_ptr()  # noqa: E731
    tokens = torch.full((rows,), -7, dtype=torch.int32, device=DEVICE)
    need = N.call("evo_hip_sample_workspace_bytes", rows, vocab) if workspace else 0
    scratch = torch.full((max(need, 16),), 255, dtype=torch.uint8, device=DEVICE)
    N.call("evo_hip_sample", CODES[logits.dtype], logits.data_ptr(), rows, vocab, logits.stride(0),
           ptr(temperature), ptr(top_k), ptr(top_p), ptr(min_p), uniform.data_ptr(),
           tokens.data_ptr(), scratch.data_ptr() if need else None, need,
           torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    return tokens.cpu()


def exact(logits, uniform, temperature, top_k, top_p, min_p):
    """One row, float64, from the definition."""
    order = np.argsort(-logits, kind="stable")
    if temperature == 0 or top_k == 1:
        return int(order[0])
    if top_k:
        order = order[:top_k]
    weight = np.exp((logits[order] - logits[order[0]]) / temperature)
    if top_p < 1:
        before = np.concatenate([[0.0], np.cumsum(weight)[:-1]])
        keep = int((before < top_p * weight.sum()).sum())
        order, weight = order[:keep], weight[:keep]
    keep = int((weight >= min_p).sum())
    order, weight = order[:keep], weight[:keep]
    ahead = np.cumsum(weight)
    return int(order[min(int(np.searchsorted(ahead, uniform * ahead[-1], side="right")),
                         keep - 1)])


def f32(values):
    return torch.tensor(values, dtype=torch.float32, device=DEVICE)


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def compare(logits, uniform, temperature, top_k, top_p, min_p, **how):
    got = sample(logits, f32(uniform), f32(temperature), i32(top_k), f32(top_p), f32(min_p), **how)
    values = logits.double().cpu().numpy()
    single = lambda x: np.float32(x).astype(np.float64)  # noqa: E731
    expected = [exact(values[r], single(uniform[r]), single(temperature[r]), top_k[r],
                      single(top_p[r]), single(min_p[r])) for r in range(len(values))]
    assert got.tolist() == expected


def parameters(rng, rows, vocab):
    """Every kind of cut alone and together."""
    uniform = rng.random(rows).astype(np.float32).tolist()
    temperature = rng.uniform(0.3, 1.7, rows).tolist()
    top_k = [int(rng.integers(1, vocab + 1)) if r % 2 else 0 for r in range(rows)]
    top_p = [float(rng.uniform(0.05, 0.999)) if r // 2 % 2 else 1.0 for r in range(rows)]
    min_p = [float(rng.uniform(0.0, 0.3)) if r // 4 % 2 else 0.0 for r in range(rows)]
    return uniform, temperature, top_k, top_p, min_p


@pytest.mark.parametrize("vocab,rows", [(1, 3), (2, 40), (3, 40), (63, 40), (64, 40), (65, 40),
                                        (512, 200), (1000, 24), (1024, 24), (1025, 24),
                                        (5000, 24), (16384, 16), (16385, 16), (50001, 16),
                                        (131072, 16), (2 ** 20, 8)])
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("workspace", [True, False])
def test_tokens(vocab, rows, kind, workspace):
    rng = np.random.default_rng(vocab)
    logits = torch.from_numpy(rng.normal(0, 2.5, (rows, vocab)).astype(np.float32))
    compare(logits.to(DEVICE).to(kind), *parameters(rng, rows, vocab), workspace=workspace)


@pytest.mark.parametrize("vocab,rows", [(8192, 257), (8193, 20), (8193, 257), (20000, 300),
                                        (65536, 257), (65537, 257)])
def test_many_rows(vocab, rows):
    """More rows than the chip has CUs, which run in smaller blocks, with ties among
    them: few bits of a logit."""
    rng = np.random.default_rng(rows * vocab)
    logits = (np.round(rng.normal(0, 2.5, (rows, vocab)) * 64) / 64).astype(np.float32)
    compare(torch.from_numpy(logits).to(DEVICE), *parameters(rng, rows, vocab))


@pytest.mark.parametrize("vocab", [512, 3000, 40000])
@pytest.mark.parametrize("workspace", [True, False])
def test_equal_logits(vocab, workspace):
    """Rows of one value, of a few, and signed zeros: ties go by index in every cut."""
    rng = np.random.default_rng(vocab)
    rows = 24
    logits = rng.integers(0, 3, (rows, vocab)).astype(np.float32)
    logits[:8] = 1.25
    logits[8:12] = np.where(rng.random((4, vocab)) < 0.5, -0.0, 0.0)
    compare(torch.from_numpy(logits).to(DEVICE), *parameters(rng, rows, vocab),
            workspace=workspace)


@pytest.mark.parametrize("vocab", [512, 20000])
def test_masked_and_extreme_logits(vocab):
    rng = np.random.default_rng(5)
    rows = 32
    logits = rng.normal(0, 2, (rows, vocab)).astype(np.float32)
    hidden = rng.random((rows, vocab)) < 0.9
    logits[:8][hidden[:8]] = -math.inf
    logits[8:16][hidden[8:16]] = np.finfo(np.float32).min
    logits[16:20] *= 1e30
    logits[20] = np.finfo(np.float32).min
    logits[21] = -math.inf
    logits[21, vocab // 2] = -1e30
    logits[22, 3] = np.finfo(np.float32).max
    logits[23] = 1e-30 * logits[23]
    compare(torch.from_numpy(logits).to(DEVICE), *parameters(rng, rows, vocab))


@pytest.mark.parametrize("vocab", [512, 20000])
def test_temperatures(vocab):
    """From nearly greedy to flat, and 0."""
    rng = np.random.default_rng(6)
    values = [0.0, 1e-38, 1e-20, 1e-4, 0.01, 0.1, 1.0, 10.0, 100.0, 1e6, 1e20, 3e38]
    rows = 2 * len(values)
    logits = rng.normal(0, 2.5, (rows, vocab)).astype(np.float32)
    uniform, _, top_k, top_p, min_p = parameters(rng, rows, vocab)
    compare(torch.from_numpy(logits).to(DEVICE), uniform, values + values, top_k, top_p, min_p)


def test_edges_of_the_draw():
    rng = np.random.default_rng(7)
    logits = torch.from_numpy(rng.normal(0, 1, (6, 512)).astype(np.float32)).to(DEVICE)
    inside = [0.0, 1e-30, 0.5, float(np.nextafter(np.float32(1), np.float32(0))), 0.25, 0.75]
    compare(logits, inside, [1.0] * 6, [0, 5, 2, 0, 512, 10000], [1.0, 1.0, 1e-9, 1.0, 0.5, 1.0],
            [0.0, 0.0, 0.0, 0.0, 1.0, 1.0])
    got = sample(logits, f32([-3.0, 0.0, 1.0, 7.0, math.inf, -math.inf]),
                 top_k=i32([4, 4, 4, 4, 4, 4]))
    order = logits.argsort(1, descending=True).cpu()
    assert got.tolist() == [int(order[r, 0 if r in (0, 1, 5) else 3]) for r in range(6)]


def test_rows_that_cannot_be_sampled():
    rng = np.random.default_rng(8)
    logits = torch.from_numpy(rng.normal(0, 1, (16, 700)).astype(np.float32)).to(DEVICE)
    one, half = [1.0] * 16, [0.5] * 16
    logits[0, 699], logits[1, 0], logits[2] = math.nan, math.inf, -math.inf
    temperature, top_k, top_p, min_p = list(one), [0] * 16, list(one), [0.0] * 16
    uniform = list(half)
    temperature[3], temperature[4], temperature[5] = -1.0, math.nan, math.inf
    top_k[6] = -1
    top_p[7], top_p[8], top_p[9] = 0.0, 1.5, math.nan
    min_p[10], min_p[11], min_p[12] = -0.1, 1.5, math.nan
    uniform[13] = math.nan
    got = sample(logits, f32(uniform), f32(temperature), i32(top_k), f32(top_p), f32(min_p))
    assert got[:14].tolist() == [NONE] * 14
    assert (got[14:] >= 0).all()


def test_defaults_and_strides():
    """NULL parameters, and rows inside a wider tensor that start anywhere."""
    rng = np.random.default_rng(9)
    for kind in (torch.float32, torch.bfloat16):
        wide = torch.from_numpy(rng.normal(0, 2, (40, 523)).astype(np.float32)).to(DEVICE).to(kind)
        logits = wide[:, 3:515]
        uniform = rng.random(40).astype(np.float32).tolist()
        got = sample(logits, f32(uniform))
        values = logits.double().cpu().numpy()
        assert got.tolist() == [exact(values[r], float(np.float32(uniform[r])), 1.0, 0, 1.0, 0.0)
                                for r in range(40)]


def test_captured_rows_split_over_blocks():
    """A large vocabulary in a graph, on a stream of its own: each replay samples the
    logits and parameters it finds, like the eager call."""
    rng = np.random.default_rng(11)
    rows, vocab = 3, 70000
    need = N.call("evo_hip_sample_workspace_bytes", rows, vocab)
    assert need > 0
    logits = torch.zeros(rows, vocab, dtype=torch.bfloat16, device=DEVICE)
    values = [f32([0.0] * rows) for _ in range(4)]  # uniform, temperature, top_p, min_p
    top_k, tokens = i32([0] * rows), i32([0] * rows)
    scratch = torch.full((need,), 255, dtype=torch.uint8, device=DEVICE)

    def draw(stream):
        N.call("evo_hip_sample", CODES[logits.dtype], logits.data_ptr(), rows, vocab, vocab,
               values[1].data_ptr(), top_k.data_ptr(), values[2].data_ptr(),
               values[3].data_ptr(), values[0].data_ptr(), tokens.data_ptr(),
               scratch.data_ptr(), need, stream.cuda_stream)

    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        draw(stream)
    for _ in range(5):
        logits.copy_(torch.from_numpy(rng.normal(0, 3, (rows, vocab)).astype(np.float32)))
        given = parameters(rng, rows, vocab)
        for to, value in zip((values[0], values[1], top_k, values[2], values[3]), given):
            to.copy_(torch.tensor(value))
        graph.replay()
        torch.cuda.synchronize()
        replayed = tokens.cpu()
        compare(logits, *given)
        draw(torch.cuda.current_stream())
        torch.cuda.synchronize()
        assert torch.equal(replayed, tokens.cpu())


def test_same_tokens_as_the_host_sampler():
    """evo_sampler_sample's token, for the draw that its generator makes."""
    import ctypes
    import os

    from evo_hip import capi
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    library = capi.EvoLibrary(os.path.join(root, "evo.cpp_amd", "lib", "libevo_hip.so"))
    lib = library.lib
    rng = np.random.default_rng(10)
    logits = rng.normal(0, 2, (60, 512)).astype(np.float32)
    top_k = [(0, 4, 100)[i % 3] for i in range(60)]
    top_p = [(1.0, 0.9, 0.5)[i // 3 % 3] for i in range(60)]
    expected, uniform = [], []
    for i in range(60):
        params = lib.evo_sampler_default_params()
        params.temperature, params.top_k, params.top_p, params.seed = 0.8, top_k[i], top_p[i], i
        sampler, token = ctypes.c_void_p(), ctypes.c_uint32()
        assert lib.evo_sampler_create(ctypes.byref(params), ctypes.byref(sampler)) == 0
        assert lib.evo_sampler_sample(
            sampler, logits[i].ctypes.data_as(ctypes.POINTER(ctypes.c_float)), 512,
            ctypes.byref(token)) == 0
        lib.evo_sampler_free(sampler)
        expected.append(token.value)
        uniform.append(np.float32(mt19937_64(i) * 2.0 ** -53))
    got = sample(torch.from_numpy(logits).to(DEVICE), f32(uniform), f32([0.8] * 60), i32(top_k),
                 f32(top_p))
    assert got.tolist() == expected


def mt19937_64(seed):
    """First output of the 64-bit Mersenne twister (Matsumoto and Nishimura), its top 53 bits."""
    mask, n, m = 2 ** 64 - 1, 312, 156
    state = [seed]
    for i in range(1, n):
        state.append((6364136223846793005 * (state[-1] ^ (state[-1] >> 62)) + i) & mask)
    x = (state[0] & 0xFFFFFFFF80000000) | (state[1] & 0x7FFFFFFF)
    y = state[m] ^ (x >> 1) ^ (0xB5026F5AA96619E9 if x & 1 else 0)
    y ^= (y >> 29) & 0x5555555555555555
    y ^= (y << 17) & 0x71D67FFFEDA60000
    y ^= (y << 37) & 0xFFF7EEE000000000
    y ^= y >> 43
    return (y & mask) >> 11


@pytest.mark.parametrize("vocab,least,most", [(512, 5, 10), (1000, 6, 11), (5000, 8, 14),
                                              (131072, 20, 27), (2 ** 20, 22, 28)])
@pytest.mark.parametrize("workspace", [True, False])
def test_draws_in_a_flat_tail(vocab, least, most, workspace):
    """One token and many equal ones far below it, and draws among those. A weight is held to
    2^-(B+1) of the largest, B = min(51, 63 - ceil(log2(vocab))): the cumulative weights on
    both sides of the token pass the draw but for vocab times that, in the running weight and
    in the total each, and for the definition's own sums in 64 bits (vocab additions of 2^-53
    of a total that is below 2, four times)."""
    rng = np.random.default_rng(vocab)
    rows = 40
    below = np.linspace(least, most, rows).astype(np.float32)
    leader = rng.integers(0, vocab, rows)
    logits = np.repeat(-below[:, None], vocab, 1)
    logits[np.arange(rows), leader] = 0.0
    weight = np.exp(-below.astype(np.float64))
    total = 1.0 + weight * (vocab - 1)
    # Steps of 2^-24 below 1 that lie in the tail.
    steps = np.maximum(1, np.floor(rng.random(rows) * (1 - 1 / total) * 2 ** 24))
    uniform = (1.0 - steps * 2.0 ** -24).astype(np.float32)
    got = sample(torch.from_numpy(logits).to(DEVICE), f32(uniform.tolist()),
                 workspace=workspace).numpy()
    bits = min(51, 63 - math.ceil(math.log2(vocab)))
    room = 2 * vocab * 2.0 ** -(bits + 1) + vocab * 2.0 ** -51
    rank = np.where(got == leader, 0, np.where(got < leader, got + 1, got))
    drawn = uniform.astype(np.float64) * total
    assert (rank > 0).all()
    assert (1.0 + (rank - 1) * weight <= drawn + room).all()
    assert (1.0 + rank * weight >= drawn - room).all()


@pytest.mark.parametrize("vocab", [512, 5000, 50257, 131072])
def test_draws_beside_borders(vocab):
    """The two F32 draws nearest to the end of a token's share, one before it and one not:
    that token and the next. (They are no nearer than the borders are held, in the definition's
    64-bit sums too.)"""
    rng = np.random.default_rng(vocab + 1)
    rows = 64
    logits = rng.normal(0, 2.5, (rows, vocab)).astype(np.float32)
    bits = min(51, 63 - math.ceil(math.log2(vocab)))
    uniform, expected = [], []
    for r in range(rows):
        order = np.argsort(-logits[r], kind="stable")
        share = np.exp(logits[r, order].astype(np.float64) - float(logits[r, order[0]]))
        total = share.sum()
        ahead = np.cumsum(share) / total
        room = vocab * (2.0 ** -bits + 2.0 ** -51)  # of the weight before the draw and the total
        # A token early in the order: its neighbours' shares are wider than F32's steps.
        rank = int(rng.integers(0, min(60, vocab // 8)))
        near = np.float32(ahead[rank])
        step = np.float32(np.inf if r % 2 else -np.inf)
        while (near >= ahead[rank]) != (r % 2 == 1) or abs(near - ahead[rank]) * total < room:
            near = np.nextafter(near, step)
        uniform.append(float(near))
        expected.append(int(order[rank + r % 2]))
    got = sample(torch.from_numpy(logits).to(DEVICE), f32(uniform))
    assert got.tolist() == expected


@pytest.mark.parametrize("vocab,rows", [(1500, 64), (20000, 16), (70000, 4)])
def test_logits_that_change_meanwhile(vocab, rows):
    """Another stream writes the logits while the call runs, flat, steep, equal and masked ones
    in turn: it ends, and gives tokens of the vocabulary or none. What is written before a
    call alone is sampled as ever."""
    rng = np.random.default_rng(vocab)
    flat = rng.normal(0, 0.1, (rows, vocab))
    steep = rng.normal(0, 30.0, (rows, vocab))
    equal = np.zeros((rows, vocab))
    masked = np.where(rng.random((rows, vocab)) < 0.99, -math.inf, 1.0)
    kinds = [torch.from_numpy(x.astype(np.float32)).to(DEVICE)
             for x in (flat, steep, equal, masked)]
    logits = kinds[0].clone()
    given = parameters(rng, rows, vocab)
    single = [f32(given[0]), f32(given[1]), i32(given[2]), f32(given[3]), f32(given[4])]
    other = torch.cuda.Stream()
    torch.cuda.synchronize()
    for i in range(12):
        with torch.cuda.stream(other):
            for j in range(6):
                logits.copy_(kinds[(i + j) % 4])
        got = sample(logits, *single, workspace=bool(i % 2))
        assert ((got == NONE) | ((got >= 0) & (got < vocab))).all()
    logits.copy_(kinds[1])
    compare(logits, *given)
