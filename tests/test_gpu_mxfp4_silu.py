"""silu(gate) * up of the 4-bit product where the sigmoid saturates: gates from -200 to 200, with up values of any size, against 64 bits."""
import pytest
import torch

import ascend_kernel_b200 as ak
from tests import mxfp4_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
LEVELS = R.E2M1
SCALES = (32.0, 8.0, 2.0, 0.5)  # of the four blocks of k of a gate column


def _codes(value):
    """Codes of four terms, a block each, that add up to about ``value`` (each the largest that still fits)."""
    left, codes = abs(value), []
    for s in SCALES:
        c = max(i for i, v in enumerate(LEVELS) if v * s <= left)
        left -= LEVELS[c] * s
        codes.append(c + (8 if value < 0 else 0))
    return codes


def _problem(rows, blocks):
    """x: rows of one value in each of four blocks of k.  ``blocks``: (gates, exponent of up) of every 32 columns of the result."""
    I = 32 * len(blocks)
    w = torch.zeros(1, 2 * I, 64, dtype=torch.uint8)
    ws = torch.zeros(1, 2 * I, 4, dtype=torch.uint8)
    for b, (gates, power) in enumerate(blocks):
        for i in range(32):
            n = 32 * b + i
            for j, c in enumerate(_codes(gates[i % len(gates)])):
                w[0, n, 16 * j] = c
                ws[0, n, j] = 127 + int(torch.log2(torch.tensor(SCALES[j])))
            w[0, I + n, 0] = (i % 7 + 1) + (8 if i % 3 == 0 else 0)  # (up: one term)
            ws[0, I + n, 0] = 127 + power
    x = torch.zeros(len(rows), 64, dtype=torch.uint8)
    for r, code in enumerate(rows):
        x[r, ::16] = code
    xs = torch.full((len(rows), 4), 127, dtype=torch.uint8)
    return x.to(DEV), xs.to(DEV), w.to(DEV), ws.to(DEV), I


def _run(x, xs, w, ws, I):
    M = x.shape[0]
    out, scale = torch.full((M, I // 2), 0x5A, dtype=torch.uint8, device=DEV), torch.full((M, I // 32), 77, dtype=torch.uint8, device=DEV)
    ak.grouped_gemm_mxfp4(x, xs, w, ws, torch.tensor([M], device=DEV), out, output_scale=scale, group_list_type=1, gate_up_silu=True)
    ak.check_status()
    return out, scale


def _check(x, xs, w, ws, I, out, scale):
    """Gates and ups are exact in fp32.  The exponential's argument is rounded, 2^-24 of |g|, and some roundings of the operations follow; what
    falls below the smallest normal number on the way is off by 2^-126 at most, times a factor below 1."""
    y = R.values(x, xs) @ R.values(w[0], ws[0]).T
    g, u = y[:, :I], y[:, I:]
    h = g * torch.sigmoid(g) * u
    assert float(h.abs().max()) < 2.0 ** 120
    eh = 16 * 2.0 ** -23 * (1 + g.abs()) * h.abs() + 2.0 ** -125
    M = x.shape[0]
    unit = torch.exp2(scale.double() - 127)
    hb, eb = h.view(M, -1, 32), eh.view(M, -1, 32)
    top, etop = hb.abs().amax(dim=2), eb.amax(dim=2)
    assert bool((scale != 255).all())
    assert bool((top - etop <= 7 * unit).all())
    assert bool(((top + etop > 3.5 * unit) | (scale == 27)).all())
    v = R.values(out, scale).view_as(hb)
    q = (hb.abs() + eb) / unit.unsqueeze(2)
    half = torch.where(q < 2, 0.25, torch.where(q < 4, 0.5, 1.0)) * unit.unsqueeze(2)
    assert bool(((v - hb).abs() <= eb + half).all())
    return top


ROWS = [2, 10, 3, 11, 1, 9, 0, 2, 4]  # 1, -1, 1.5, -1.5, 0.5, -0.5, 0, 1, 2
NEAR = [[c + 0.25 * i for i in range(8)] for c in (-130.0, -104.0, -91.0, -89.0, -88.0, -87.0, -86.0, -81.0, -80.0, -79.5, -30.0, -5.0, -1.0, 0.0, 1.0, 20.0, 88.0, 129.0)]


@pytest.mark.parametrize("power", [0, 20, 40, 60, 90, 104])
def test_gates_where_the_sigmoid_saturates(power):
    """Blocks whose 32 gates lie side by side, so that none of them hides behind a larger one."""
    blocks = [(g, power) for g in NEAR]
    blocks += [([0.5], 0)] * (-len(blocks) % 4)
    # (rows of 1.5 and 2 take the gates to +-260 and the ups along with them)
    args = _problem(ROWS, blocks)
    top = _check(*args, *_run(*args))
    if power >= 60:  # the tail is there to be lost: non-zero results of gates below -87
        tail = [b for b, g in enumerate(NEAR) if max(g) < -87]
        assert bool((top[0, tail] >= 2.0 ** -98).any())


def test_saturated_gates_beside_ordinary_ones():
    """One column of 32 far down the tail, the others ordinary: the ordinary ones have the bits that they have without it."""
    plain = _problem(ROWS, [([0.5, -2.0, 3.25, -7.5], 0)] * 4)
    x, xs, w, ws, I = _problem(ROWS, [([0.5, -2.0, 3.25, -7.5], 0)] * 4)
    for n in range(5, I, 32):
        for j, c in enumerate(_codes(-100.0)):
            w[0, n, 16 * j] = c
    a, b = _run(*plain), _run(x, xs, w, ws, I)
    _check(x, xs, w, ws, I, *b)
    rows = [0, 2, 4]  # (positive rows: the replaced column is all but zero there and was no block's largest)
    va, vb = R.values(a[0], a[1]).view(len(ROWS), -1, 32), R.values(b[0], b[1]).view(len(ROWS), -1, 32)
    keep = [i for i in range(32) if i != 5]
    assert torch.equal(a[1][rows], b[1][rows]) and torch.equal(va[rows][:, :, keep], vb[rows][:, :, keep])


@pytest.mark.parametrize("M", [1, 15, 17, 40, 97, 130, 192, 193, 400])
def test_every_number_of_pieces(M):
    """Tiles of 16 to 192 rows with the tail in some of them."""
    gen = torch.Generator().manual_seed(M)
    rows = [ROWS[i] for i in torch.randint(0, len(ROWS), (M,), generator=gen).tolist()]
    blocks = [(NEAR[i], p) for i, p in ((0, 90), (2, 60), (4, 60), (13, 0), (10, 40), (6, 100), (15, 0), (5, 70))]
    args = _problem(rows, blocks)
    _check(*args, *_run(*args))


def test_infinite_sums_stay_not_finite():
    """A gate or an up that overflows fp32 gives its block the scale NaN, also where the other is far down the tail."""
    x, xs, w, ws, I = _problem([2, 2], [([-100.0], 0), ([1.0], 0), ([1.0], 0), ([1.0], 0)])
    xs[1] = 254
    ws[0, I + 3, 0] = 250  # row 1: 2^127 * 2^123 * code
    out, scale = _run(x, xs, w, ws, I)
    assert int(scale[1, 0]) == 255 and bool((out[1, :16] == 0).all()) and int(scale[0, 1]) != 255


def test_tail_tiles_among_others_again_and_again():
    """Tiles whose buffer goes back late between ones whose does at once: several experts, one of which has gates far down, and the same bits each time."""
    gen = torch.Generator(device=DEV).manual_seed(3)
    counts, K, I = [200, 30, 0, 500, 97], 256, 1024
    M, G = sum(counts), len(counts)
    x = torch.randint(0, 256, (M, K // 2), generator=gen, device=DEV).to(torch.uint8)
    xs = torch.randint(122, 124, (M, K // 32), generator=gen, device=DEV).to(torch.uint8)
    xs = torch.nn.functional.pad(xs, (0, R.width(K) - K // 32))
    w = torch.randint(0, 256, (G, 2 * I, K // 2), generator=gen, device=DEV).to(torch.uint8)
    ws = torch.randint(122, 124, (G, 2 * I, R.width(K)), generator=gen, device=DEV).to(torch.uint8)
    ws[1], ws[3, 32:64] = 129, 130  # (gates of some hundreds)
    ws[3, I + 32:I + 64] = 190
    gl = torch.tensor(counts, dtype=torch.int64, device=DEV)

    def run():
        out, scale = torch.full((M, I // 2), 0x5A, dtype=torch.uint8, device=DEV), torch.full((M, I // 32), 77, dtype=torch.uint8, device=DEV)
        ak.grouped_gemm_mxfp4(x, xs, w, ws, gl, out, output_scale=scale, group_list_type=1, gate_up_silu=True)
        return out, scale

    first = run()
    a = 0
    for g, c in enumerate(counts):
        if c:
            _check(x[a:a + c], xs[a:a + c], w[g:g + 1], ws[g:g + 1], I, first[0][a:a + c], first[1][a:a + c])
        a += c
    for _ in range(20):
        for p, q in zip(run(), first):
            assert torch.equal(p, q)
    ak.check_status()
