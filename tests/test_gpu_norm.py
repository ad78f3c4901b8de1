"""GPU parity of the norms of rows (larder_amd.trunk.norm_rows, read_codes) with float64.

Tolerances: half a step of the result's type (finfo.eps / 2 of the value), and of float32 arithmetic, u = 2^-24: the sum of squares
of h channels is off by less than (h / lanes + 12) u of itself (one chain a lane, at most 12 additions of a tree), its root by
half of that and 3 u, the sum of two rows by u of their magnitudes and the three products by u each. (h / 256 < 80 here for rows
in registers; longer ones have a chain of h / 32.)"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
U = 2.0 ** -24
# below the type's normal numbers a step is absolute
TINY = {F16: 2.0 ** -25, BF16: 2.0 ** -134, F32: 2.0 ** -150}


def host(t):
    return t.detach().double().cpu().numpy()


def normal(gen, *shape, dtype=BF16, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def norm(x, r, w, eps):
    s = host(x) + (host(r) if r is not None else 0.0)
    y = s / np.sqrt((s * s).mean(-1, keepdims=True) + eps) * host(w)
    size = np.abs(host(x)) + (np.abs(host(r)) if r is not None else 0.0)
    # what an error of `size` u in s makes of y, in the value itself and through the row's mean square
    spread = U * size * np.abs(host(w)) / np.sqrt((s * s).mean(-1, keepdims=True) + eps)
    chain = (x.shape[-1] / 256 + 12) / 2 + 3 + 5
    return s, y, spread + np.abs(y) * U * (chain + (size ** 2).sum(-1, keepdims=True) / ((s * s).sum(-1, keepdims=True) + 1e-300))


def check(x, r, w, eps, **kw):
    from larder_amd import trunk
    got = trunk.norm_rows(x, w, eps, residual=r, **kw)
    s, y, loose = norm(x, r, w, eps)
    if r is not None:
        got, total = got[:-1], got[-1]
        want = host(total)
        size = np.abs(host(x)) + np.abs(host(r))
        assert (np.abs(want - s) <= torch.finfo(x.dtype).eps / 2 * np.abs(s) * (1 + U) + U * size + TINY[x.dtype]).all()
        got = got[0] if len(got) == 1 else got
    if kw.get("group"):
        codes, scales = got
        g = kw["group"]
        assert codes.dtype is torch.float8_e4m3fn and codes.shape == x.shape
        assert scales.shape == x.shape[:-1] + (x.shape[-1] // g,) and scales.dtype is F32
        sc = host(scales)[..., None]
        parts, tol = y.reshape(*sc.shape[:-1], g), loose.reshape(*sc.shape[:-1], g)
        most, off = np.abs(parts).max(-1, keepdims=True), tol.max(-1, keepdims=True)
        # the least power of two, of a largest magnitude within the tolerance
        assert (np.frexp(sc)[0] == 0.5).all() and (sc >= 2.0 ** -100).all()
        assert (most <= 448 * sc + off).all() and ((most >= 224 * sc - off) | (sc == 2.0 ** -100)).all()
        # half a step of e4m3 (2^-4 of the value; 2^-10 below its normal numbers)
        back = trunk.read_codes(codes, scales, F32)
        bar = tol + np.maximum(2.0 ** -4 * (np.abs(parts) + tol), 2.0 ** -10 * sc)
        assert (np.abs(host(back).reshape(parts.shape) - parts) <= bar).all()
        # bfloat16 holds code times scale, unless it is below its normal numbers
        assert torch.equal(trunk.read_codes(codes, scales).float(), back.to(BF16).float())
    else:
        assert got.dtype is x.dtype and got.shape == x.shape and got.is_contiguous()
        eps_t = torch.finfo(x.dtype).eps / 2
        assert (np.abs(host(got) - y) <= eps_t * np.abs(y) + (1 + eps_t) * loose + TINY[x.dtype]).all()


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("t,h", [(1, 1), (3, 7), (1, 64), (33, 65), (5, 100), (300, 128), (2, 255), (70, 512), (9, 513), (1, 2048),
                                 (17, 2051), (4, 4096), (3, 5000), (2, 8191), (3, 16384), (2, 16385), (1, 20001),
                                 (2048, 513), (2300, 1024), (2049, 1100), (2050, 1536)])
def test_norm(dtype, t, h):
    gen = torch.Generator(device="cuda").manual_seed(h)
    x, w = normal(gen, t, h, dtype=dtype) * torch.exp(normal(gen, h)).to(dtype), normal(gen, h, dtype=dtype)
    check(x, None, w, 1e-6)
    r = normal(gen, t, h, dtype=dtype, scale=3.0)
    check(x, r, w.float(), 1e-5)
    check(x, r, w, 1e-6, group=h)
    check(x, None, w, 1e-6, group=h)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("t,h,group", [(1, 64, 32), (7, 96, 32), (5, 512, 64), (3, 640, 128), (40, 2048, 128), (2, 4096, 256),
                                       (3, 1024, 512), (2, 16384, 128), (2, 16512, 32), (1, 17408, 512), (9, 192, 64)])
def test_groups(dtype, t, h, group):
    gen = torch.Generator(device="cuda").manual_seed(h + group)
    x = normal(gen, t, h, dtype=dtype) * torch.exp(normal(gen, h)).to(dtype)
    x[-1, :group] = 0
    check(x, None, normal(gen, h, dtype=dtype), 1e-6, group=group)
    r = normal(gen, t, h, dtype=dtype)
    r[-1, :group] = 0
    check(x, r, normal(gen, h, dtype=F32), 1e-6, group=group)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("h", [64, 128, 256, 100])
def test_heads_of_a_product(dtype, h):
    """Views: the heads of q and k among a product's outputs, rows of odd offsets, one row, many axes."""
    from larder_amd import trunk
    gen = torch.Generator(device="cuda").manual_seed(h)
    whole = normal(gen, 37, 9, h, dtype=dtype)
    w = normal(gen, h, dtype=dtype)
    check(whole[:, 2:7], None, w, 1e-6)
    check(whole[::3, ::2], None, w, 1e-6)
    flat = normal(gen, 12 * (h + 3) + 1, dtype=dtype)
    check(flat[1:1 + 12 * (h + 3)].view(12, h + 3)[:, 1:1 + h], None, w, 1e-6)
    check(flat[5:5 + h], None, w, 1e-6)
    check(whole.view(37, 3, 3, h), None, w, 1e-6)
    check(whole.transpose(0, 1), normal(gen, 9, 37, h, dtype=dtype), w, 1e-6)
    last = whole.transpose(1, 2)[..., :8]  # an axis that is not dense
    check(last, None, normal(gen, 8, dtype=dtype), 1e-6)
    assert trunk.norm_rows(whole[:0], w).shape == (0, 9, h)
    assert trunk.norm_rows(whole[:, :0], w, residual=whole[:, :0])[1].shape == (37, 0, h)


@pytest.mark.parametrize("h", [40, 512, 4096, 16388])
@pytest.mark.parametrize("where", ["residual", "x", "view"])
def test_sum_in_place(h, where):
    from larder_amd import trunk
    gen = torch.Generator(device="cuda").manual_seed(h)
    x, r, w = normal(gen, 11, h), normal(gen, 11, h), normal(gen, h)
    y, s = trunk.norm_rows(x, w, residual=r)
    codes = trunk.norm_rows(x, w, residual=r, group=h)
    for group in (None, h):
        a, b = x.clone(), r.clone()
        room = normal(gen, 13, h + 5)
        kept, total = room.clone(), {"residual": b, "x": a, "view": room[1:12, 3:3 + h]}[where]
        got = trunk.norm_rows(a, w, residual=b, group=group, total=total)
        assert got[-1] is total and torch.equal(total, s)
        assert torch.equal(got[0].view(torch.uint8), (y if group is None else codes[0]).view(torch.uint8))
        if where == "view":
            room[1:12, 3:3 + h] = kept[1:12, 3:3 + h]
            assert torch.equal(room, kept)
    # without a residual: the sum is x
    z = torch.empty_like(x)
    assert torch.equal(trunk.norm_rows(x, w, total=z)[0], trunk.norm_rows(x, w)) and torch.equal(z, x)


@pytest.mark.parametrize("h", [48, 512, 2000, 16400])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_large_small_and_not_finite(h, dtype):
    """Squares that pass float32; rows of zeros; infinities and NaN, which stay in their rows."""
    from larder_amd import trunk
    gen = torch.Generator(device="cuda").manual_seed(h)
    x, w = normal(gen, 9, h, dtype=dtype), normal(gen, h, dtype=dtype)
    x[0] *= 2.0 ** 66
    x[1] *= 2.0 ** 120
    x[2] *= 2.0 ** -100
    x[3] = 0
    check(x, None, w, 1e-6)
    check(x, -x.flip(0), w, 1e-6)
    x[5, h // 2] = float("inf")
    x[7, 3] = float("nan")
    y = trunk.norm_rows(x, w)
    s, want, loose = norm(x[[0, 1, 2, 3, 4, 6, 8]], None, w, 1e-6)
    assert (np.abs(host(y[[0, 1, 2, 3, 4, 6, 8]]) - want) <= torch.finfo(dtype).eps * (np.abs(want) + loose) + loose + TINY[dtype]).all()
    assert torch.isnan(y[7]).all() and torch.isnan(y[5, h // 2])
    rest = torch.arange(h, device="cuda") != h // 2
    assert (y[5][rest] == 0).all()
    codes, scales = trunk.norm_rows(x, w, group=h)
    assert (codes[7].view(torch.uint8) & 0x7f).eq(0x7f).all() and scales[7, 0] == 2.0 ** -100
    assert codes[5].view(torch.uint8)[h // 2] & 0x7f == 0x7f and (codes[5].float()[rest] == 0).all()
    assert scales[3, 0] == 2.0 ** -100 and (codes[3].float() == 0).all()


def test_read_codes():
    from larder_amd import trunk
    gen = torch.Generator(device="cuda").manual_seed(1)
    for t, h, g in ((1, 1, 1), (3, 7, 7), (5, 24, 3), (9, 100, 25), (4, 4096, 128), (2, 10, 5), (1000, 333, 333)):
        codes = torch.randint(0, 256, (t, h), dtype=torch.uint8, generator=gen, device="cuda").view(torch.float8_e4m3fn)
        scales = torch.exp2(torch.randint(-20, 20, (t, h // g), generator=gen, device="cuda").float())
        want = (codes.double().view(t, h // g, g) * scales.double()[..., None]).view(t, h)
        for dtype in (F16, BF16, F32):
            got = trunk.read_codes(codes, scales, dtype)
            assert torch.equal(got.view(t, h).nan_to_num(5e4), want.float().to(dtype).nan_to_num(5e4))
        assert torch.equal(trunk.read_codes(codes.view(-1)[:h], scales[0], F32).nan_to_num(), want[0].float().nan_to_num())


def test_norm_in_a_graph_and_on_a_stream():
    from larder_amd import trunk
    gen = torch.Generator(device="cuda").manual_seed(2)
    x, r, w = normal(gen, 40, 2048), normal(gen, 40, 2048), normal(gen, 2048)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        trunk.norm_rows(x, w, residual=r)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, s = trunk.norm_rows(x, w, residual=r)
        c = trunk.norm_rows(s, w, group=128)
    for turn in range(4):
        x.copy_(normal(gen, 40, 2048))
        r.copy_(normal(gen, 40, 2048))
        graph.replay()
        torch.cuda.synchronize()
        y2, s2 = trunk.norm_rows(x, w, residual=r)
        c2 = trunk.norm_rows(s2, w, group=128)
        assert torch.equal(y, y2) and torch.equal(s, s2) and torch.equal(c[1], c2[1])
        assert torch.equal(c[0].view(torch.uint8), c2[0].view(torch.uint8))


def test_refusals():
    from larder_amd import trunk
    x, w = torch.zeros(3, 64, dtype=BF16, device="cuda"), torch.zeros(64, dtype=BF16, device="cuda")
    for kw, why in ((dict(weight=w[:63]), "weight"), (dict(weight=w.half()), "weight"), (dict(eps=0.0), "eps"), (dict(eps=-1.0), "eps"),
                    (dict(eps=float("nan")), "eps"), (dict(residual=x[:2]), "residual"), (dict(residual=x.half()), "residual"),
                    (dict(group=48), "48 channels"), (dict(group=128), "128 channels"), (dict(group=0), "0 channels"),
                    (dict(total=x.half()), "total"), (dict(total=x.t().contiguous().t()), "total"), (dict(total=x[0]), "total"),
                    (dict(residual=x.cpu()), "devices"), (dict(x=x.long(), weight=w.float()), "dtype"), (dict(x=x[:, :0]), "channels")):
        with pytest.raises(ValueError, match=why):
            trunk.norm_rows(**{**dict(x=x, weight=w), **kw})
    codes, scales = trunk.norm_rows(x, w, group=32)
    for args, why in (((codes.float(), scales), "codes"), ((codes, scales[:2]), "scales"), ((codes, scales.half()), "scales"),
                      ((codes[:, :63], scales), "scales"), ((codes, scales, torch.int32), "dtype"), ((codes, scales.cpu()), "devices")):
        with pytest.raises(ValueError, match=why):
            trunk.read_codes(*args)
