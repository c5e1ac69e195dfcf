"""Rotary positions in their general form against a 64-bit rotation by complex numbers."""
import pytest
import torch

from dhellam_amd.operators.rope import rotary_bwd, rotary_frequencies, rotary_fwd, rotary_table

pytestmark = pytest.mark.gpu

PARTS = {"kind": "parts", "factor": 16.0, "original_length": 4096}
BANDS = {"kind": "bands", "factor": 8.0, "original_length": 8192}


def turned(x, theta, rot, interleaved, scaling, positions, backward=False):
    f, factor = rotary_frequencies(theta, rot, scaling)
    angle = positions.double()[:, None] * torch.tensor(f, dtype=torch.float64, device=x.device)
    w = torch.polar(torch.full_like(angle, factor), -angle if backward else angle)[:, None, :]
    y = x.double().clone()
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    z = torch.complex(y[..., a].contiguous(), y[..., b].contiguous()) * w
    size = torch.zeros_like(y)
    size[..., a] = size[..., b] = x.double()[..., a].abs() + x.double()[..., b].abs()
    y[..., a], y[..., b] = z.real, z.imag
    return y, size * factor


def check(got, x, *args, **kw):
    """A rounding to the type, and cos / sin that are off by 2^-17 (16 bits; hardware instructions on an angle good to 2^-25 turns) or, in
    fp32, by half a step each of the angle, the series' last addition, the factor, two products and their sum: 6 2^-24; exact elsewhere."""
    want, size = turned(x, *args, **kw)
    eps = torch.finfo(x.dtype).eps
    slack = 6 * 2.0 ** -24 if x.dtype == torch.float32 else 2.0 ** -17
    bound = (want.abs() + slack * size) * eps / 2 + slack * size + torch.finfo(x.dtype).smallest_normal
    assert ((got.double() - want).abs() <= bound).all(), ((got.double() - want).abs() / bound).max()
    rot = args[1]
    assert torch.equal(got[..., rot:], x[..., rot:])


def rand(*shape, dtype, seed=0):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens,hq,hk,d,rot", [
    (1, 1, 1, 2, 2), (1, 32, 8, 128, 128), (7, 8, 1, 128, 64), (33, 3, 2, 80, 20), (5, 4, 4, 100, 50), (3, 2, 1, 13, 6), (64, 12, 4, 96, 96),
    (300, 5, 5, 72, 18), (1000, 8, 1, 256, 256), (2, 130, 3, 64, 32), (9, 0, 2, 64, 64), (17, 1, 0, 65, 64),
    (130, 3, 2, 128, 64), (64, 5, 1, 192, 128), (201, 7, 3, 64, 32), (4100, 9, 0, 64, 64), (63, 1, 1, 40, 6)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_forward_and_backward(tokens, hq, hk, d, rot, interleaved, dtype):
    q, k = rand(tokens, hq, d, dtype=dtype), rand(tokens, hk, d, dtype=dtype, seed=1)
    at = torch.randint(0, 5000, (tokens,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(2), dtype=torch.int32)
    t = rotary_table(10000.0, rot, "cuda", interleaved)
    args = (10000.0, rot, interleaved, None, at)
    for turn, back in ((rotary_fwd, False), (rotary_bwd, True)):
        qo, ko, ms = turn(q, k, t, at)
        assert ms == 0 and qo.is_contiguous() and qo.dtype == dtype
        check(qo, q, *args, backward=back)
        check(ko, k, *args, backward=back)


@pytest.mark.parametrize("scaling", [None, {"kind": "linear", "factor": 4.0}, {"kind": "ntk", "factor": 8.0}, PARTS, BANDS])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_far_positions_and_scaled_frequencies(scaling, dtype):
    """Positions past 2^20, 2^24 and 2^31, and before zero: 64-bit angles of 2^40 are good to 2^-53 2^40 = 2^-13 of a turn, so the 64-bit
    form is only asked up to 2^24; past it whole numbers are."""
    t = rotary_table(500000.0, 128, "cuda", False, scaling)
    base = torch.tensor([0, 1, 4095, 131071, (1 << 20) + 3, (1 << 24) - 1, -1, -70000], device="cuda")
    q, k = rand(8, 4, 128, dtype=dtype), rand(8, 2, 128, dtype=dtype, seed=1)
    for at in (base, base.to(torch.int32)):
        qo, ko, _ = rotary_fwd(q, k, t, at)
        check(qo, q, 500000.0, 128, False, scaling, base)
        check(ko, k, 500000.0, 128, False, scaling, base)
    # whole numbers: the turn of position p + 2^64 / step is a whole one, so far positions have near twins
    steps = [u % 2 ** 64 for u in t.steps.tolist()]
    far = (1 << 40) + 12345
    one = torch.tensor([far], device="cuda")
    got, _, _ = rotary_fwd(q[:1], None, t, one)
    angle = torch.tensor([(far * u % 2 ** 64) / 2.0 ** 64 for u in steps], dtype=torch.float64) * 2 * torch.pi
    w = torch.polar(torch.full_like(angle, t.factor), angle).cuda()
    z = torch.complex(q[:1, :, :64].double(), q[:1, :, 64:].double()) * w
    want, size = torch.cat((z.real, z.imag), -1), (q[:1, :, :64].double().abs() + q[:1, :, 64:].double().abs()).repeat(1, 1, 2) * t.factor
    slack = 6 * 2.0 ** -24 if dtype == torch.float32 else 2.0 ** -17
    assert ((got.double() - want).abs() <= want.abs() * torch.finfo(dtype).eps / 2 + 1.01 * slack * size).all()


@pytest.mark.parametrize("tokens,seq_len", [(1, None), (100, None), (100, 32), (100, 1)])
def test_positions_by_default(tokens, seq_len):
    t = rotary_table(10000.0, 32, "cuda", True)
    q = rand(tokens, 2, 64, dtype=torch.float16)
    at = torch.arange(tokens, device="cuda") % (seq_len or tokens)
    qo, ko, _ = rotary_fwd(q, None, t, None, seq_len)
    assert ko is None
    check(qo, q, 10000.0, 32, True, None, at)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_parts_and_in_place(interleaved, dtype):
    """Views of a packed projection, heads first, a part in the middle of the head, odd offsets; in place what surrounds them stays."""
    t = rotary_table(10000.0, 24, "cuda", interleaved)
    at = torch.arange(11, device="cuda") * 7
    packed = rand(11, 3 * 64 + 2 * 64 + 3, dtype=dtype)
    views = lambda p: (p[:, 1:193].unflatten(1, (3, 64)), p[:, 193:321].unflatten(1, (2, 64)))
    q, k = views(packed)
    qo, ko, _ = rotary_fwd(q, k, t, at)
    check(qo, q, 10000.0, 24, interleaved, None, at)
    check(ko, k, 10000.0, 24, interleaved, None, at)
    there = packed.clone()
    a, b, _ = rotary_fwd(*views(there), t, at, inplace=True)
    assert a.data_ptr() == views(there)[0].data_ptr() and torch.equal(a, qo) and torch.equal(b, ko)
    assert torch.equal(there[:, 0], packed[:, 0]) and torch.equal(there[:, 321:], packed[:, 321:])
    heads_first = rand(3, 11, 64, dtype=dtype)                       # [heads, tokens, d]
    ho, _, _ = rotary_fwd(heads_first.transpose(0, 1), None, t, at)
    check(ho, heads_first.transpose(0, 1), 10000.0, 24, interleaved, None, at)
    part = rand(11, 4, 64, dtype=dtype)
    kept = part.clone()
    rotary_fwd(part[..., 40:], None, t, at, inplace=True)
    assert torch.equal(part[..., :40], kept[..., :40])
    check(part[..., 40:], kept[..., 40:], 10000.0, 24, interleaved, None, at)
    one = rand(1, 1, 64, dtype=dtype).expand(11, 4, 64)              # a broadcast input is read, not written
    eo, _, _ = rotary_fwd(one, None, t, at)
    check(eo, one.contiguous(), 10000.0, 24, interleaved, None, at)


def test_backward_is_the_transpose_and_undoes_the_forward():
    t = rotary_table(10000.0, 64, "cuda", False, PARTS)
    at = torch.arange(50, device="cuda") * 997
    q, g = rand(50, 4, 96, dtype=torch.float32), rand(50, 4, 96, dtype=torch.float32, seed=3)
    y, dx = rotary_fwd(q, None, t, at)[0], rotary_bwd(g, None, t, at)[0]
    a, b = (y.double() * g.double()).sum(), (q.double() * dx.double()).sum()
    assert abs(a - b) <= 1e-6 * (y.double().norm() * g.double().norm())
    back = rotary_bwd(y, None, t, at)[0]
    # two turns of 6 2^-24 (|a| + |b|) each, |a| + |b| up to sqrt 2 of the pair's length, and the factor squared
    want = q.double().clone()
    want[..., :64] *= t.factor ** 2
    assert (back.double() - want).abs().max() <= 24 * 2.0 ** -24 * t.factor ** 2 * q.abs().max()


def test_values_that_are_not_finite_stay_in_their_pair():
    t = rotary_table(10000.0, 32, "cuda")
    q = rand(6, 2, 64, dtype=torch.bfloat16)
    at = torch.arange(6, device="cuda")
    want = rotary_fwd(q, None, t, at)[0]
    bad = q.clone()
    bad[3, 1, 5], bad[4, 0, 40] = torch.nan, torch.inf
    got = rotary_fwd(bad, None, t, at)[0]
    changed = torch.zeros_like(q, dtype=torch.bool)
    changed[3, 1, [5, 21]] = True
    changed[4, 0, 40] = True
    assert torch.equal(got[~changed], want[~changed]) and got[3, 1, 5].isnan() and got[4, 0, 40].isinf()


def test_another_stream_and_replays_of_a_graph():
    t = rotary_table(10000.0, 128, "cuda")
    q, k = rand(257, 8, 128, dtype=torch.bfloat16), rand(257, 1, 128, dtype=torch.bfloat16, seed=1)
    want = rotary_fwd(q, k, t)[:2]
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    got = rotary_fwd(q, k, t, stream=st, profiling=True)
    torch.cuda.synchronize()
    assert got[2] > 0 and torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rotary_fwd(q, k, t)[:2]
    for i in range(3):
        q.copy_(rand(257, 8, 128, dtype=torch.bfloat16, seed=10 + i))
        graph.replay()
        torch.cuda.synchronize()
        want = rotary_fwd(q, k, t)[:2]
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_more_lanes_than_one_launch():
    """2^30 + 70 tokens of two heads of two elements: two launches, positions past 2^30, addresses past 2^32."""
    n = (1 << 30) + 70
    t = rotary_table(10000.0, 2, "cuda")
    q = torch.empty(n, 2, 2, dtype=torch.bfloat16, device="cuda")
    q.view(-1).view(torch.int64).fill_(0x3F8040003F804040)                # four ordinary values
    ends = [slice(0, 100), slice((1 << 30) - 30, (1 << 30) + 70)]
    rows = [q[s].clone() for s in ends]
    rotary_fwd(q, None, t, inplace=True)
    for s, x in zip(ends, rows):
        check(q[s], x, 10000.0, 2, False, None, torch.arange(s.start, s.stop, device="cuda"))


def test_one_of_the_two_in_place():
    """The C entry takes q in place and k not: every element of both is turned once, also where a part is no whole number of pieces."""
    from dhellam_amd import _lib
    t, at = rotary_table(10000.0, 20, "cuda"), torch.arange(70, device="cuda", dtype=torch.int32)
    q, k = rand(70, 3, 41, dtype=torch.float16), rand(70, 2, 41, dtype=torch.float16, seed=1)
    want = rotary_fwd(q, k, t, at)[:2]
    a, b = q.clone(), torch.full_like(k, 7.0)
    call = lambda head: _lib.load().dh_rotary(a.data_ptr(), k.data_ptr(), a.data_ptr(), b.data_ptr(), t.steps.data_ptr(), at.data_ptr(), 4, 70, 3, 2, 41, 20,
                                              123, 41, 82, 41, 123, head, 82, 41, 0, 0, 0, 1.0, 2, torch.cuda.current_stream().cuda_stream)
    _lib.check(call(41))
    assert torch.equal(a, want[0]) and torch.equal(b, want[1])
    assert call(42) == -1 and "strides" in _lib.load().dh_last_error().decode()


def test_refusals():
    t = rotary_table(10000.0, 32, "cuda")
    q, k = rand(4, 2, 64, dtype=torch.float16), rand(4, 1, 64, dtype=torch.float16)
    at = torch.arange(4, device="cuda")
    for bad in [lambda: rotary_fwd(q[..., :16], None, t), lambda: rotary_fwd(q, k.float(), t), lambda: rotary_fwd(q, k[:3], t),
                lambda: rotary_fwd(q, k, t, at.float()), lambda: rotary_fwd(q, k, t, at[:3]), lambda: rotary_fwd(q, k, t, None, -1),
                lambda: rotary_fwd(q[0], k[0], t), lambda: rotary_fwd(q.transpose(1, 2), None, t), lambda: rotary_fwd(q, q, t, inplace=True),
                lambda: rotary_fwd(q[:1].expand(4, 2, 64), None, t, inplace=True), lambda: rotary_fwd(q[:, :1].expand(4, 2, 64), None, t, inplace=True),
                lambda: rotary_fwd(q.as_strided((4, 2, 64), (64, 32, 1)), None, t, inplace=True)]:
        with pytest.raises(AssertionError):
            bad()
    for bad in [lambda: rotary_fwd(q.double(), None, t), lambda: rotary_fwd(q, k.cpu(), t), lambda: rotary_fwd(q, k, t, at.cpu()),
                lambda: rotary_fwd(q, k, rotary_table(10000.0, 32, "cpu")), lambda: rotary_fwd(q, k, t, stream=7)]:
        with pytest.raises(RuntimeError):
            bad()
    assert rotary_fwd(q[:0], k[:0], t)[0].shape == (0, 2, 64)


@pytest.mark.parametrize("tokens,hq,hk,d,rot,dtype", [
    (14003, 32, 8, 128, 128, torch.bfloat16), (7001, 31, 10, 256, 128, torch.float16), (7003, 33, 8, 128, 64, torch.float32),      # past the caches
    (6001, 9, 2, 64, 32, torch.bfloat16), (3001, 7, 4, 192, 64, torch.float16), (3001, 7, 4, 64, 32, torch.float32),               # a rest, in groups of 64 tokens
    (4001, 7, 4, 80, 20, torch.float16), (9001, 5, 0, 72, 18, torch.bfloat16), (5003, 3, 4, 41, 6, torch.float32)])                # a rest, by single tokens
@pytest.mark.parametrize("interleaved", [False, True])
def test_many_tokens(tokens, hq, hk, d, rot, dtype, interleaved):
    """Enough of them for two heads a lane, odd numbers of heads among them; beside the tensors and over views of a packed projection."""
    t = rotary_table(10000.0, rot, "cuda", interleaved)
    at = torch.randint(0, 5000, (tokens,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    packed = rand(tokens, (hq + hk + 1) * d, dtype=dtype)
    views = lambda p: (p[:, :hq * d].unflatten(1, (hq, d)), p[:, hq * d:(hq + hk) * d].unflatten(1, (hk, d)) if hk else None)
    q, k = views(packed)
    args = (10000.0, rot, interleaved, None, at)
    for turn, back in ((rotary_fwd, False), (rotary_bwd, True)):
        qo, ko, _ = turn(q, k, t, at)
        check(qo, q, *args, backward=back)
        if hk:
            check(ko, k, *args, backward=back)
        there = packed.clone()
        a, b, _ = turn(*views(there), t, at, inplace=True)
        assert torch.equal(a, qo) and (hk == 0 or torch.equal(b, ko))
        assert torch.equal(there[:, (hq + hk) * d:], packed[:, (hq + hk) * d:])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hq,hk,d,rot", [(7, 4, 80, 20), (8, 1, 128, 128), (6, 2, 64, 40), (12, 4, 96, 48)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_a_token_is_the_same_in_every_call(hq, hk, d, rot, interleaved, dtype):
    """Alone, among a few and among many, in place and not: the same bits, every time."""
    t = rotary_table(10000.0, rot, "cuda", interleaved, PARTS)
    at = torch.arange(9001, device="cuda") * 11
    q, k = rand(9001, hq, d, dtype=dtype), rand(9001, hk, d, dtype=dtype, seed=1)
    qo, ko, _ = rotary_fwd(q, k, t, at)
    for _ in range(3):
        again = rotary_fwd(q, k, t, at)
        assert torch.equal(again[0], qo) and torch.equal(again[1], ko)
    for s in (slice(0, 1), slice(17, 150), slice(8000, 9001)):
        a, b, _ = rotary_fwd(q[s], k[s], t, at[s])
        assert torch.equal(a, qo[s]) and torch.equal(b, ko[s])
    rotary_fwd(q, k, t, at, inplace=True)
    assert torch.equal(q, qo) and torch.equal(k, ko)
