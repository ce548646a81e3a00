"""The 8-bit cache's kernels against their definition in 64 bits (plain_kv8)."""
import math

import pytest
import torch

import plain_kv8 as plain
from esp_b200.csrc import ops
from esp_b200.errors import Backend
from esp_b200.parts.base import Workspace

pytestmark = pytest.mark.gpu
PAGE, BAD_INDEX = 64, 8
E4M3 = torch.float8_e4m3fn


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def pools(pages, nkv, hd, seed=None):
    """Codes of keys and values and exponents; with a seed rows of ordinary size, else bytes that no kernel may use (NaN)."""
    if seed is None:
        k, v = (torch.full((pages, nkv, PAGE, hd), 0x7F, dtype=torch.uint8, device="cuda").view(E4M3) for _ in range(2))
        return k, v, torch.full((pages, nkv, 2, PAGE), 255, dtype=torch.uint8, device="cuda")
    g = gen(seed)
    out, exps = [], torch.empty((pages, nkv, 2, PAGE), dtype=torch.uint8, device="cuda")
    for which in range(2):
        x = torch.randn((pages, nkv, PAGE, hd), generator=g, device="cuda") * torch.exp(torch.randn((pages, nkv, PAGE, 1), generator=g, device="cuda"))
        if which == 0:
            x[..., 3 % hd] *= 8
        codes, e = plain.quantize(x.double())
        out.append(codes.float().to(E4M3))
        exps[:, :, which] = (e + 127).to(torch.uint8)
    return out[0], out[1], exps


def tables(lengths, seed, spare=3):
    """Pages of the sequences in no order, -1 behind each sequence's last: (table, number of pages)."""
    need = [(n + PAGE - 1) // PAGE for n in lengths]
    total = sum(need) + spare
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    t, at = torch.full((len(lengths), max(need) + 1), -1, dtype=torch.int32), 0
    for i, n in enumerate(need):
        t[i, :n] = order[at:at + n]
        at += n
    return t.cuda(), total


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def status():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


def sequence_rows(pool, exps, which, pages, length):
    """float64 [nkv, length, hd] of a sequence's rows."""
    x = plain.stored(pool[pages], exps[pages, :, which])
    return x.transpose(0, 1).flatten(1, 2)[:, :length]


# ------------------------------------------------------------------------------------------------------- append
APPEND = [
    # nh, nkv, hd, rot, news, pasts, bias
    (16, 16, 128, 128, [1], [0], True),
    (16, 16, 128, 128, [1], [63], False),
    (4, 2, 16, 16, [1, 1, 1], [5, 64, 127], True),
    (5, 5, 24, 24, [3, 70], [62, 1], True),
    (7, 1, 80, 40, [130], [17], False),
    (6, 3, 96, 0, [9, 1], [120, 0], True),
    (28, 4, 128, 128, [1] * 67, list(range(40, 107)), True),
    (4, 4, 64, 64, [200, 1, 66], [0, 300, 62], False),
    (2, 1, 192, 192, [65], [10], True),
    (8, 8, 256, 256, [33, 40], [50, 0], True),
    (3, 3, 256, 128, [5], [59], False),
    (1, 1, 8, 4, [2], [0], False),
]


@pytest.mark.parametrize("nh,nkv,hd,rot,news,pasts,with_bias", APPEND)
def test_append(nh, nkv, hd, rot, news, pasts, with_bias):
    n, width = sum(news), (nh + 2 * nkv) * hd
    g = gen(n + hd)
    table, total = tables([a + b for a, b in zip(news, pasts)], 7)
    k, v, exps = pools(total, nkv, hd, seed=n)
    before = [t.clone() for t in (k.view(torch.uint8), v.view(torch.uint8), exps)]
    qkv = torch.randn((n, width), generator=g, device="cuda") * torch.exp(2 * torch.randn((n, 1), generator=g, device="cuda"))
    bias = torch.randn(width, generator=g, device="cuda") if with_bias else None
    most = max(a + b for a, b in zip(news, pasts))
    angle = torch.arange(most, device="cuda")[:, None] * 1e4 ** (-torch.arange(rot // 2, device="cuda") / max(1, rot // 2))
    cos, sin = angle.cos().contiguous(), angle.sin().contiguous()
    seq = ints([i for i, t in enumerate(news) for _ in range(t)])
    pos = ints([p + j for p, t in zip(pasts, news) for j in range(t)])
    q, st = torch.empty((n, nh * hd), dtype=torch.bfloat16, device="cuda"), status()
    ops.kv8_rope_append(qkv, bias, seq, pos, cos, sin, rot, q, k, v, exps, table, PAGE, nh, nkv, hd, True, st)
    assert st.item() == 0
    x = (qkv.double() + (bias.double() if with_bias else 0)).view(n, nh + 2 * nkv, hd)
    turned, big = x.clone(), x.abs()
    if rot:
        c, s = cos.double()[pos.long()], sin.double()[pos.long()]
        turned[:, :nh + nkv] = plain.rotate(x[:, :nh + nkv], c, s, rot)
        h = rot // 2
        both = big[:, :nh + nkv, :h] + big[:, :nh + nkv, h:rot]
        big[:, :nh + nkv, :rot] = torch.cat((both, both), -1)
    # 32-bit: the bias's sum, two products and their sum are each off by at most half a step, 2^-24 of the operands' size
    err = 4 * 2.0 ** -24 * (big + (bias.double().abs().max() if with_bias else 0))
    got = q.double().view(n, nh, hd)
    assert torch.all((got - turned[:, :nh]).abs() <= 2.0 ** -8 * turned[:, :nh].abs() + 2 * err[:, :nh])
    page, place = table[seq.long(), (pos // PAGE).long()].long(), (pos % PAGE).long()
    for pool, which, lo in ((k, 0, nh), (v, 1, nh + nkv)):
        want, e64 = turned[:, lo:lo + nkv], plain.row_exponent(turned[:, lo:lo + nkv].abs().amax(-1))
        e = exps[page, :, which, place].double() - 127
        slack = err[:, lo:lo + nkv].amax(-1)
        top = want.abs().amax(-1)
        # the exponent of the definition, or the one of a maximum that rounding may have moved over a border
        assert torch.all((e == plain.row_exponent(top + slack)) | (e == plain.row_exponent((top - slack).clamp_min(0))))
        assert (e == e64).double().mean() > 0.99
        rows = plain.stored(pool[page, :, place], exps[page, :, which, place])
        # half a step of e4m3: 2^-4 of the number, or half of 2^(e - 9) below the normal range
        half_step = torch.maximum(2.0 ** -4 * want.abs(), torch.exp2(e - 10)[..., None])
        assert torch.all((rows - want).abs() <= half_step + 2 * err[:, lo:lo + nkv])
        if not rot and not with_bias or (which == 1 and not with_bias):
            codes, _ = plain.quantize(want)
            assert torch.equal(pool[page, :, place].double(), codes)
    # nothing else has changed
    touched = torch.zeros((total, PAGE), dtype=torch.bool, device="cuda")
    touched[page, place] = True
    for t, old in zip((k.view(torch.uint8), v.view(torch.uint8)), before):
        assert torch.equal(t.transpose(1, 2)[~touched], old.transpose(1, 2)[~touched])
    assert torch.equal(exps.permute(0, 3, 1, 2)[~touched], before[2].permute(0, 3, 1, 2)[~touched])


@pytest.mark.parametrize("nh,nkv,hd,rot,news,pasts,with_bias", [
    (6, 2, 80, 20, [9, 3], [62, 0], True),
    (5, 5, 104, 100, [3], [127], True),
    (3, 1, 256, 250, [5, 1], [60, 300], True),
    (2, 2, 64, 2, [70], [1], False),
    (7, 1, 128, 126, [300, 33], [0, 64], True),
    (1, 1, 40, 34, [1], [0], True),
])
def test_append_of_rotations_that_are_no_multiple_of_eight(nh, nkv, hd, rot, news, pasts, with_bias):
    """The kernel whose lanes hold every 32nd number: rotation partners in other slices, more heads than a block has warps."""
    test_append(nh, nkv, hd, rot, news, pasts, with_bias)


@pytest.mark.parametrize("hd,rot", [(128, 128), (128, 0), (80, 40), (256, 256), (64, 0)])
def test_append_of_rows_at_the_borders(hd, rot):
    """Maxima at and beside 448 * 2^e, ties, subnormal codes, zeros, the smallest and largest exponents, rows that are no numbers.
    Position 0: the rotation is by an angle of zero, so numbers arrive as they are."""
    rows = []
    for e in (-100, -37, 0, 5, 100):
        s = 2.0 ** e
        rows += [[448 * s], [448 * (1 + 2.0 ** -23) * s, 1.0 * s], [-448 * s, 2.0 ** -9 * s, 2.0 ** -10 * s, 3 * 2.0 ** -10 * s, -5 * 2.0 ** -10 * s],
                 [240 * s, 17 * s, 17.5 * s, 18 * s, 19 * s, 1.0625 * s, 1.1875 * s], [448.1 * s, -0.0]]
    rows += [[0.0], [1e-45], [-1e-38, 3e-39], [2.0 ** -101 * 448], [math.inf], [1.0, -math.inf], [math.nan, 3.0], [3e38], [-0.0]]
    n = len(rows)
    x = torch.zeros((n, 3, hd), device="cuda")
    for i, r in enumerate(rows):
        x[i, 1, :len(r)] = torch.tensor(r)
        x[i, 2, hd - len(r):] = torch.tensor(r)
        if rot and not all(map(math.isfinite, r)):         # infinity times the sine 0 is not a number either way
            x[i, 1] = 0
    k, v, exps = pools(n, 1, hd)
    cos, sin = torch.ones((1, rot // 2), device="cuda"), torch.zeros((1, rot // 2), device="cuda")
    q = torch.empty((n, hd), dtype=torch.bfloat16, device="cuda")
    table, st = torch.arange(n, dtype=torch.int32, device="cuda")[:, None].contiguous(), status()
    ops.kv8_rope_append(x.view(n, -1), None, torch.arange(n, dtype=torch.int32, device="cuda"), ints([0] * n), cos, sin, rot, q, k, v, exps,
                        table, PAGE, 1, 1, hd, True, st)
    assert st.item() == 0
    for pool, which in ((k, 0), (v, 1)):
        codes, e = plain.quantize(x[:, 1 + which].double())
        byte = torch.where(torch.isnan(e), 255.0, e + 127)
        assert torch.equal(exps[:, 0, which, 0].double(), byte)
        assert torch.equal(pool[:, 0, 0].double(), codes)


def test_append_of_queries_alone_and_bad_places():
    nh, nkv, hd = 4, 2, 64
    qkv = torch.randn((5, (nh + 2 * nkv) * hd), generator=gen(1), device="cuda")
    cos, sin = torch.ones((200, 32), device="cuda"), torch.zeros((200, 32), device="cuda")
    k, v, exps = pools(3, nkv, hd)
    q, st = torch.zeros((5, nh * hd), dtype=torch.bfloat16, device="cuda"), status()
    seq, pos = ints([0, 0, 1, 1, 1]), ints([0, 1, 64, 65, 3])
    ops.kv8_rope_append(qkv, None, seq, pos, cos, sin, hd, q, None, None, None, None, PAGE, nh, nkv, hd, False, st)
    assert st.item() == 0
    assert torch.equal(q, qkv[:, :nh * hd].to(torch.bfloat16))
    # sequence 2 is not in the table
    ops.kv8_rope_append(qkv[:1], None, ints([2]), ints([1]), cos, sin, hd, q[:1], k, v, exps, ints([[0], [1]]), PAGE, nh, nkv, hd, True, st)
    assert st.item() == BAD_INDEX and (exps == 255).all()
    # page 7 and page -1 are not there, position 200 has no angle, position 130 no entry of the table, -1 is no position
    table = ints([[2, 0], [7, -1]])
    for where in ([3, 0, 2, 2, 2], [3, 70, 0, 100, 2]):
        st.zero_()
        for t in (k.view(torch.uint8), v.view(torch.uint8), exps):
            t.fill_(255)
        ops.kv8_rope_append(qkv, None, ints([0, 0, 1, 1, 0]), ints([where[0], 64, where[2], 70, [200, 130][where[1] != 0]]), cos, sin, hd, q, k, v, exps,
                            table, PAGE, nh, nkv, hd, True, st)
        assert st.item() == BAD_INDEX
        written = (exps[:, 0, 0] != 255).nonzero().tolist()
        assert written == sorted([[2, 3], [0, 0]])
    ops.kv8_rope_append(qkv[:1], None, ints([0]), ints([-1]), cos, sin, hd, q[:1], k, v, exps, table, PAGE, nh, nkv, hd, True, st)
    assert st.item() == BAD_INDEX


# ------------------------------------------------------------------------------------------------------- attention
def check_rows(got, want, spread, q, k, hd, weight_step):
    """|got - want| <= half a step of bfloat16 of the result, plus what rounding the weights (half a step of their type) and the
    errors of the scores (twice: numerator and sum) and of exp2 (2^-21) may move it."""
    nan = torch.isnan(want)
    assert torch.equal(nan, torch.isnan(got))
    slack = weight_step + 2 * plain.score_error(q, k, hd) + 2.0 ** -20
    bound = 2.0 ** -8 * want.abs() + (1 + 2.0 ** -8) * slack * spread + 1e-38
    off = (got - want).abs() - bound
    assert torch.all(off[~nan] <= 0), f"off by {float((got - want)[~nan].abs().max())}, {float(off[~nan].max())} over the bound"


DECODE = [
    # nh, nkv, hd, lengths (the new token among them), window
    (1, 1, 128, [1], 0),
    (16, 16, 128, [1, 2, 31, 32, 33, 63, 64, 65], 0),
    (16, 16, 128, [777], 0),
    (28, 4, 128, [1000, 129, 4097], 0),
    (12, 1, 128, [300, 5], 0),
    (16, 1, 64, [513], 0),
    (34, 2, 64, [129, 640], 0),
    (40, 2, 128, [200], 0),
    (4, 2, 16, [70, 3], 0),
    (5, 5, 24, [150], 70),
    (7, 7, 80, [99, 260], 0),
    (6, 2, 104, [130], 64),
    (8, 2, 192, [385, 64], 0),
    (3, 3, 256, [200, 1], 0),
    (20, 2, 256, [333], 100),
    (4, 4, 64, [1, 5, 64, 65, 700, 1400], 1),
    (4, 4, 64, [1, 5, 64, 65, 700, 1400], 64),
    (8, 4, 128, [2000, 40], 333),
    (2, 1, 128, [20000], 0),
    (2, 1, 128, [20000, 300], 5000),
    (16, 16, 128, [130] * 40, 0),
    (2, 2, 128, [3000, 1, 129, 128, 127, 5000] * 5, 0),
    (1, 1, 64, [70 + 13 * i for i in range(1100)], 0),
    (24, 2, 96, [1, 95, 96, 97, 1500], 0),
    (7, 7, 96, [2000, 31, 640], 100),
    (3, 3, 72, [129, 4000], 0),
    (16, 1, 88, [900], 0),
    # enough keys for blocks of sixteen rows
    (12, 1, 128, [40000, 33000, 50000, 1], 0),
    (28, 2, 72, [30000, 25001, 20000], 0),
    (34, 2, 104, [30000, 25001, 20000], 20000),
    (2, 1, 8, [300], 0),
]


def decode_inputs(nh, nkv, hd, lengths, seed):
    table, total = tables(lengths, seed)
    k, v, exps = pools(total, nkv, hd, seed)
    n = len(lengths)
    q = (torch.randn((n, nh * hd), generator=gen(seed + 1), device="cuda") * 2).to(torch.bfloat16)
    return table, k, v, exps, q, torch.arange(n, dtype=torch.int32, device="cuda"), ints([length - 1 for length in lengths])


def check_decode(out, q, k, v, exps, table, lengths, nh, hd, window):
    for i, length in enumerate(lengths):
        pages = table[i, :(length + PAGE - 1) // PAGE].long()
        kk, vv = (sequence_rows(p, exps, w, pages, length) for p, w in ((k, 0), (v, 1)))
        qq = q[i].double().view(1, nh, hd)
        want, spread = plain.attend(qq, kk, vv, torch.tensor([length - 1], device="cuda"), window)
        check_rows(out[i].double().view(1, nh, hd), want, spread, qq, kk, hd, 2.0 ** -11)


@pytest.mark.parametrize("nh,nkv,hd,lengths,window", DECODE)
def test_decode(nh, nkv, hd, lengths, window):
    table, k, v, exps, q, seq, pos = decode_inputs(nh, nkv, hd, lengths, 11)
    out, st, ws = torch.full_like(q, math.nan), status(), Workspace(q.device)
    for _ in range(2):                              # the second call finds the counters as the first one left them
        out.fill_(math.nan)
        ops.attn_decode_kv8(q, k, v, exps, out, ws, seq, pos, table, PAGE, nh, nkv, hd, window, st)
        assert st.item() == 0
        check_decode(out, q, k, v, exps, table, lengths, nh, hd, window)
    # keys that were cached long before: the same bits
    again = torch.empty_like(out)
    ops.attn_decode_kv8(q, k, v, exps, again, ws, seq, pos, table, PAGE, nh, nkv, hd, window, st, seq_past=ints([length - 1 for length in lengths]))
    assert torch.equal(out, again)


@pytest.mark.parametrize("nh,nkv,hd", [(28, 2, 72), (18, 2, 96), (32, 2, 104), (20, 2, 128)])
@pytest.mark.parametrize("lengths,window", [([30000, 25001, 20000, 35000], 0), ([30000, 25001, 20000, 35000], 33333), ([9000, 1, 8000, 700] * 5, 500)])
def test_decode_of_more_than_eight_heads_on_one(nh, nkv, hd, lengths, window):
    """With far to go a block takes sixteen rows, with a short window eight, whatever the page table's width."""
    table, k, v, exps, q, seq, pos = decode_inputs(nh, nkv, hd, lengths, 13)
    out, st = torch.full_like(q, math.nan), status()
    ops.attn_decode_kv8(q, k, v, exps, out, Workspace(q.device), seq, pos, table, PAGE, nh, nkv, hd, window, st)
    assert st.item() == 0
    check_decode(out, q, k, v, exps, table, lengths, nh, hd, window)


@pytest.mark.parametrize("nh,nkv,hd", [(4, 4, 128), (12, 1, 64)])
def test_decode_with_rows_that_are_no_numbers(nh, nkv, hd):
    """NaN where the mask hides it (behind the row, ahead of its window) changes nothing; where it is seen the row is NaN."""
    lengths, window = [300, 300, 300, 300], 100
    table, k, v, exps, q, seq, pos = decode_inputs(nh, nkv, hd, lengths, 3)
    out, st, ws = torch.empty_like(q), status(), Workspace(q.device)
    ops.attn_decode_kv8(q, k, v, exps, out, ws, seq, pos, table, PAGE, nh, nkv, hd, window, st)
    for i, (at, which) in enumerate([(199, 0), (200, 0), (200, 1), (199, 1)]):
        exps[table[i, at // PAGE].long(), :, which, at % PAGE] = 255
    last = table[:, 299 // PAGE].long()               # behind the last position: bytes that are no rows
    exps[last, :, :, 300 % PAGE:] = 255
    k.view(torch.uint8)[last, :, 300 % PAGE:] = 0x7F
    v.view(torch.uint8)[last, :, 300 % PAGE:] = 0xFF
    got = torch.empty_like(q)
    ops.attn_decode_kv8(q, k, v, exps, got, ws, seq, pos, table, PAGE, nh, nkv, hd, window, st)
    assert torch.equal(got[0], out[0]) and torch.equal(got[3], out[3])
    assert torch.isnan(got[1]).all() and torch.isnan(got[2]).all()
    assert st.item() == 0


@pytest.mark.parametrize("group", [1, 12])
@pytest.mark.parametrize("key_scale,value_scale", [(2.0 ** 90, 1.0), (2.0 ** -95, 1.0), (1.0, 2.0 ** 92), (1.0, 2.0 ** -92)])
def test_decode_with_exponents_far_apart(group, key_scale, value_scale):
    """Rows whose exponents differ by far more than a half's range; queries scaled against the keys."""
    hd, length = 64, 500
    g = gen(5)
    x = torch.randn((2, length, hd), generator=g, device="cuda", dtype=torch.float64)
    far = torch.arange(length, device="cuda") % 3 == 1
    x[0] *= key_scale
    x[1] *= torch.where(far, value_scale, 1.0)[:, None]
    q = (torch.randn((1, group, hd), generator=g, device="cuda").double() * 3 / key_scale).to(torch.bfloat16)
    table, total = tables([length], 2)
    k, v, exps = pools(total, 1, hd, 1)
    for which, pool in ((0, k), (1, v)):
        codes, e = plain.quantize(x[which])
        page, place = table[0, torch.arange(length, device="cuda") // PAGE].long(), torch.arange(length, device="cuda") % PAGE
        pool.view(torch.uint8)[page, 0, place] = codes.float().to(E4M3).view(torch.uint8)
        exps[page, 0, which, place] = (e + 127).to(torch.uint8)
    out, st = torch.empty_like(q), status()
    ops.attn_decode_kv8(q, k, v, exps, out, Workspace(q.device), ints([0]), ints([length - 1]), table, PAGE, group, 1, hd, 0, st)
    assert st.item() == 0
    check_decode(out, q, k, v, exps, table, [length], group, hd, 0)


def test_decode_weights_of_few_strong_and_many_weak_keys():
    """One key takes nearly all of the softmax's mass, thousands share the rest and all point the same way."""
    hd, length = 64, 9000
    table, total = tables([length], 2)
    k, v, exps = pools(total, 1, hd, 1)
    k.view(torch.uint8).zero_()
    v.view(torch.uint8).fill_(0x38)                   # 1.0
    exps.fill_(127)
    first = table[0, 0].long()
    k.view(torch.uint8)[first, 0, 0] = 0x38
    v.view(torch.uint8)[first, 0, 0] = 0
    for score in (8.0, 13.0):                         # weights of the others e^-8, e^-13 of the strong one's
        q = torch.full((1, hd), score / math.sqrt(hd), device="cuda").to(torch.bfloat16)
        out, st = torch.empty_like(q), status()
        ops.attn_decode_kv8(q, k, v, exps, out, Workspace(q.device), ints([0]), ints([length - 1]), table, PAGE, 1, 1, hd, 0, st)
        check_decode(out, q, k, v, exps, table, [length], 1, hd, 0)


def test_decode_with_pages_that_are_none():
    nh, nkv, hd, lengths = 4, 2, 128, [300, 200, 64, 100]
    table, k, v, exps, q, seq, pos = decode_inputs(nh, nkv, hd, lengths, 9)
    out, st, ws = torch.empty_like(q), status(), Workspace(q.device)
    ops.attn_decode_kv8(q, k, v, exps, out, ws, seq, pos, table, PAGE, nh, nkv, hd, 0, st)
    bad = table.clone()
    bad[1, 1], bad[2, 0], bad[3, 1] = k.shape[0], -1, -2147483648
    got = torch.empty_like(out)
    ops.attn_decode_kv8(q, k, v, exps, got, ws, seq, pos, bad, PAGE, nh, nkv, hd, 0, st)
    assert st.item() == BAD_INDEX
    assert torch.equal(got[0], out[0]) and torch.isfinite(got).all()
    assert (got[2] == 0).all()                        # not one page: no keys
    st.zero_()
    got.fill_(7)
    ops.attn_decode_kv8(q, k, v, exps, got, ws, ints([0, 1, [-1, 4][hd > 64], 3]), ints([299, -1, 63, 99 + 64 * table.shape[1]]), table, PAGE, nh, nkv, hd, 0, st)
    assert st.item() == BAD_INDEX and torch.equal(got[0], out[0]) and (got[1:] == 7).all()


def test_decode_of_a_sequence_twice_in_a_call():
    nh, nkv, hd, lengths = 8, 2, 128, [70, 700, 333]
    table, k, v, exps, q, seq, pos = decode_inputs(nh, nkv, hd, lengths, 4)
    ws, st, out = Workspace(q.device), status(), torch.empty_like(q)
    ops.attn_decode_kv8(q, k, v, exps, out, ws, seq, pos, table, PAGE, nh, nkv, hd, 0, st)
    order = [2, 0, 1, 2]
    rows, got = torch.tensor(order, device="cuda"), torch.empty((4, nh * hd), dtype=torch.bfloat16, device="cuda")
    # the same sequence twice in a call; rows in another order
    ops.attn_decode_kv8(q[rows], k, v, exps, got, ws, ints(order), pos[rows], table, PAGE, nh, nkv, hd, 0, st)
    check_decode(got[:3], q[rows[:3]], k, v, exps, table[rows[:3]], [lengths[i] for i in order[:3]], nh, hd, 0)


PREFILL = [
    # nh, nkv, hd, news, pasts, window
    (1, 1, 128, [1], [0], 0),
    (2, 2, 128, [2], [0], 0),
    (4, 4, 128, [200], [0], 0),
    (4, 2, 128, [128, 127, 129], [0, 64, 63], 0),
    (7, 1, 128, [300, 5, 1, 64], [1000, 0, 257, 128], 0),
    (4, 2, 64, [257], [130], 0),
    (2, 2, 64, [400], [100], 77),
    (3, 3, 128, [300, 33], [500, 10], 129),
    (2, 1, 128, [300], [0], 1),
    (4, 2, 16, [150], [3], 0),
    (5, 5, 24, [140, 2], [0, 70], 70),
    (2, 1, 80, [130], [65], 0),
    (3, 1, 104, [260], [0], 0),
    (2, 2, 192, [140], [30], 0),
    (2, 1, 256, [129, 20], [0, 200], 50),
    (1, 1, 128, [1500], [700], 0),
    # enough (tile, head) items that two tiles of a sequence go together
    (32, 4, 64, [1300, 700, 129, 64], [0, 333, 5, 1000], 0),
    (48, 16, 128, [1030, 400], [70, 0], 0),
    (40, 8, 128, [1700, 130, 1, 300], [200, 1000, 64, 0], 260),
    (60, 60, 104, [1281], [0], 1),
    (48, 3, 24, [900, 900], [3, 60], 1000),
    # between: the kernel looks at what the tiles see (in pairs; singly; tiles of unequal length; with a window)
    (35, 5, 128, [706], [1953], 0),
    (16, 8, 64, [2048], [0], 0),
    (7, 1, 128, [2500, 5, 1, 640], [100, 900, 0, 1], 0),
    (12, 3, 104, [1500, 300], [0, 700], 150),
    # sequences of few new tokens among longer ones, and alone
    (7, 1, 128, [300, 5, 32, 33, 1, 16, 17], [100, 3000, 64, 64, 700, 0, 127], 0),
    (24, 8, 96, [16, 17, 2, 31], [700, 65, 0, 2000], 0),
    (4, 2, 104, [32, 33, 1, 1, 1], [300, 300, 5, 64, 1000], 100),
    (5, 5, 72, [9, 3], [1000, 0], 1),
    (16, 4, 128, [1000, 7, 7, 7, 7, 7, 7, 7, 7, 7, 7, 7], [0] + [50 * i for i in range(11)], 0),
]


def prefill_inputs(nh, nkv, hd, news, pasts, seed):
    table, total = tables([a + b for a, b in zip(news, pasts)], seed)
    k, v, exps = pools(total, nkv, hd, seed)
    starts = [0]
    for t in news:
        starts.append(starts[-1] + t)
    q = (torch.randn((starts[-1], nh * hd), generator=gen(seed + 1), device="cuda") * 2).to(torch.bfloat16)
    tiles = sorted(((i, f) for i, t in enumerate(news) for f in range(0, t, 128)), key=lambda x: -(pasts[x[0]] + min(x[1] + 128, news[x[0]])))
    return table, k, v, exps, q, starts, ints([t[0] for t in tiles]), ints([t[1] for t in tiles])


def check_prefill(out, q, k, v, exps, table, starts, pasts, nh, hd, window):
    for i, past in enumerate(pasts):
        a, b = starts[i], starts[i + 1]
        length = past + b - a
        pages = table[i, :(length + PAGE - 1) // PAGE].long()
        kk, vv = (sequence_rows(p, exps, w, pages, length) for p, w in ((k, 0), (v, 1)))
        qq = q[a:b].double().view(b - a, nh, hd)
        want, spread = plain.attend(qq, kk, vv, torch.arange(past, length, device="cuda"), window)
        check_rows(out[a:b].double().view(b - a, nh, hd), want, spread, qq, kk, hd, 2.0 ** -8)


@pytest.mark.parametrize("nh,nkv,hd,news,pasts,window", PREFILL)
def test_prefill(nh, nkv, hd, news, pasts, window):
    table, k, v, exps, q, starts, tile_seq, tile_first = prefill_inputs(nh, nkv, hd, news, pasts, 21)
    out, st = torch.full_like(q, math.nan), status()
    for _ in range(2):
        out.fill_(math.nan)
        ops.attn_prefill_kv8(q, k, v, exps, out, tile_seq, tile_first, ints(starts), ints(pasts), table, PAGE, nh, nkv, hd, window, st)
        assert st.item() == 0
        check_prefill(out, q, k, v, exps, table, starts, pasts, nh, hd, window)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_prefill_with_rows_that_are_no_numbers(hd):
    """A position that is no number makes the rows that see it NaN, and leaves the others' bits alone: those before it, and those
    whose window has passed it."""
    nh, nkv, news, pasts, window = 4, 2, [400], [50], 150
    table, k, v, exps, q, starts, tile_seq, tile_first = prefill_inputs(nh, nkv, hd, news, pasts, 5)
    out, got, st = torch.empty_like(q), torch.empty_like(q), status()
    args = (tile_seq, tile_first, ints(starts), ints(pasts), table, PAGE, nh, nkv, hd, window, st)
    ops.attn_prefill_kv8(q, k, v, exps, out, *args)
    for which, at in ((0, 211), (1, 230)):
        kept = exps.clone()
        exps[table[0, at // PAGE].long(), 0, which, at % PAGE] = 255
        ops.attn_prefill_kv8(q, k, v, exps, got, *args)
        assert st.item() == 0
        pos = torch.arange(50, 450, device="cuda")
        sees = (pos >= at) & (pos - at < window)
        a, b = got.view(400, nh, hd), out.view(400, nh, hd)
        assert torch.isnan(a[sees][:, :2]).all()
        assert torch.equal(a[~sees], b[~sees]) and torch.equal(a[:, 2:], b[:, 2:])
        exps.copy_(kept)
    # what lies behind the last position is not looked at
    last = table[0, 449 // PAGE].long()
    exps[last, :, :, 450 % PAGE:] = 255
    k.view(torch.uint8)[last, :, 450 % PAGE:] = 0x7F
    v.view(torch.uint8)[last, :, 450 % PAGE:] = 0xFF
    ops.attn_prefill_kv8(q, k, v, exps, got, *args)
    assert torch.equal(got, out)


@pytest.mark.parametrize("hd", [128, 192])
@pytest.mark.parametrize("value_scale", [2.0 ** 92, 2.0 ** -92])
def test_prefill_with_exponents_far_apart(hd, value_scale):
    nh, nkv, news, pasts = 2, 1, [200], [100]
    table, k, v, exps, q, starts, tile_seq, tile_first = prefill_inputs(nh, nkv, hd, news, pasts, 6)
    shift = round(math.log2(value_scale))
    e = exps[:, :, 1, ::3].int() + shift
    exps[:, :, 1, ::3] = e.clamp(27, 227).to(torch.uint8)
    exps[:, :, 0] = (exps[:, :, 0].int() + 60).to(torch.uint8)
    q = (q.float() * 2.0 ** -60).to(torch.bfloat16)
    out, st = torch.empty_like(q), status()
    ops.attn_prefill_kv8(q, k, v, exps, out, tile_seq, tile_first, ints(starts), ints(pasts), table, PAGE, nh, nkv, hd, 0, st)
    check_prefill(out, q, k, v, exps, table, starts, pasts, nh, hd, 0)


@pytest.mark.parametrize("nh,hd,rise", [(2, 128, 7.5), (2, 64, 7.5), (40, 128, 7.5), (2, 192, 37.8), (2, 128, 37.8), (12, 128, 37.8), (12, 64, 37.8)])
def test_the_largest_values_behind_a_maximum_that_lags(nh, hd, rise):
    """The first 256 values have the largest exponent, and the scores of 12,000 more lie ``rise`` (in units of log2) above theirs, just below
    where a kernel would go over to a larger maximum (where that looks at weights times 2^exponent: with exponents 30 smaller).  Sums of
    unnormalised weights times values pass 32-bit's range, the result does not."""
    past, new, low = 12288 - 130, 130, 256
    table, total = tables([past + new], 2)
    k, v, exps = pools(total, 1, hd, 1)
    k.view(torch.uint8).zero_()
    k.view(torch.uint8)[..., 0] = 0x40                    # 2
    first = table[0, :low // PAGE].long()
    k.view(torch.uint8)[first] = 0
    v.view(torch.uint8).fill_(0x7D)                       # 416
    v.view(torch.uint8)[..., 1::2] = 0xFA                 # -320
    exps[:, :, 0], exps[:, :, 1] = 127, 227 if rise < 8 else 197
    exps[first, :, 1] = 227
    q = torch.zeros((new, nh, hd), device="cuda")
    q[..., 0] = rise / 2 * math.log(2) * math.sqrt(hd)
    q = q.to(torch.bfloat16).view(new, -1)
    out, one, st = torch.full_like(q, math.nan), torch.full_like(q, math.nan), status()
    args = (table, PAGE, nh, 1, hd, 0, st)
    ops.attn_prefill_kv8(q, k, v, exps, out, ints([0, 0]), ints([128, 0]), ints([0, new]), ints([past]), *args)
    ops.attn_decode_kv8(q, k, v, exps, one, Workspace(q.device), ints([0] * new), torch.arange(past, past + new, dtype=torch.int32, device="cuda"), *args)
    assert st.item() == 0
    check_prefill(out, q, k, v, exps, table, [0, new], [past], nh, hd, 0)
    check_prefill(one, q, k, v, exps, table, [0, new], [past], nh, hd, 0)


@pytest.mark.parametrize("hd", [128, 192])
def test_prefill_with_pages_that_are_none(hd):
    nh, nkv, news, pasts = 2, 1, [150, 150], [100, 30]
    table, k, v, exps, q, starts, tile_seq, tile_first = prefill_inputs(nh, nkv, hd, news, pasts, 8)
    out, got, st = torch.empty_like(q), torch.empty_like(q), status()
    ops.attn_prefill_kv8(q, k, v, exps, out, tile_seq, tile_first, ints(starts), ints(pasts), table, PAGE, nh, nkv, hd, 0, st)
    assert st.item() == 0
    bad = table.clone()
    bad[1, 1] = k.shape[0] + 5
    ops.attn_prefill_kv8(q, k, v, exps, got, tile_seq, tile_first, ints(starts), ints(pasts), bad, PAGE, nh, nkv, hd, 0, st)
    assert st.item() == BAD_INDEX
    assert torch.equal(got[:150], out[:150]) and torch.isfinite(got).all()


@pytest.mark.parametrize("nh,nkv,hd,news,pasts,window,missing", [
    # missing: (sequence, page of it)
    (4, 2, 128, [150, 150], [100, 30], 0, [(0, 1), (1, 0), (1, 2)]),
    (4, 2, 64, [300, 129], [0, 64], 0, [(0, 0), (0, 3), (1, 1)]),
    (2, 2, 104, [400], [100], 77, [(0, 2), (0, 3), (0, 6)]),
    (32, 4, 64, [1300, 700], [0, 333], 0, [(0, 0), (0, 1), (0, 9), (1, 5)]),
    (48, 16, 128, [1030, 400], [70, 0], 150, [(0, 4), (0, 5), (0, 6), (0, 7), (1, 2)]),
    (2, 2, 192, [140, 40], [30, 0], 0, [(0, 1), (1, 0)]),
    (7, 1, 128, [300, 5, 32], [100, 3000, 64], 0, [(0, 3), (1, 20), (2, 0), (2, 1)]),
])
def test_keys_of_pages_that_are_none_have_no_weight(nh, nkv, hd, news, pasts, window, missing):
    """The same in prompts as in decode: a softmax over the keys that are there, zeros where there are none."""
    table, k, v, exps, q, starts, tile_seq, tile_first = prefill_inputs(nh, nkv, hd, news, pasts, 17)
    bad, st, ws = table.clone(), status(), Workspace(q.device)
    for n, (i, page) in enumerate(missing):
        bad[i, page] = [-1, k.shape[0], 2 ** 31 - 1][n % 3]
    out, one = torch.full_like(q, math.nan), torch.full_like(q, math.nan)
    ops.attn_prefill_kv8(q, k, v, exps, out, tile_seq, tile_first, ints(starts), ints(pasts), bad, PAGE, nh, nkv, hd, window, st)
    assert st.item() == BAD_INDEX
    seq = ints([i for i, t in enumerate(news) for _ in range(t)])
    pos = ints([past + j for past, t in zip(pasts, news) for j in range(t)])
    ops.attn_decode_kv8(q, k, v, exps, one, ws, seq, pos, bad, PAGE, nh, nkv, hd, window, st)
    empty = 0
    for i, past in enumerate(pasts):
        a, b = starts[i], starts[i + 1]
        length = past + b - a
        pages = table[i, :(length + PAGE - 1) // PAGE].long()
        kk, vv = (sequence_rows(p, exps, w, pages, length) for p, w in ((k, 0), (v, 1)))
        qq = q[a:b].double().view(b - a, nh, hd)
        at = torch.arange(past, length, device="cuda")
        j = torch.arange(length, device="cuda")
        sees = (j[None] <= at[:, None]) & ((at[:, None] - j[None] < window) if window else True)
        for page in (page for s, page in missing if s == i):
            sees = sees & (j // PAGE != page)[None]
        score = torch.einsum("rhd,hld->rhl", qq, kk.repeat_interleave(nh // nkv, 0)) / math.sqrt(hd)
        p = torch.nan_to_num(torch.softmax(torch.where(sees[:, None], score, -math.inf), -1))     # a row without keys: zeros
        want, spread = (torch.einsum("rhl,hld->rhd", p, x.repeat_interleave(nh // nkv, 0)) for x in (vv, vv.abs()))
        none = ~sees.any(-1)
        empty += int(none.sum())
        for got, step in ((out, 2.0 ** -8), (one, 2.0 ** -11)):
            check_rows(got[a:b].double().view(b - a, nh, hd), want, spread, qq, kk, hd, step)
            assert (got[a:b][none] == 0).all()
    assert empty > 0


def test_an_infinite_query_among_pages_that_are_none():
    """All scores the lowest: NaN where the row has a key, zeros where it has none."""
    nh, nkv, hd, news, pasts = 2, 1, 128, [200], [0]
    table, k, v, exps, q, starts, tile_seq, tile_first = prefill_inputs(nh, nkv, hd, news, pasts, 6)
    k.view(torch.uint8)[..., 5] = 0x38
    q.view(-1, nh, hd)[[10, 70], 1, 5] = -math.inf
    table[0, 0] = -1
    out, st = torch.full_like(q, math.nan), status()
    ops.attn_prefill_kv8(q, k, v, exps, out, tile_seq, tile_first, ints(starts), ints(pasts), table, PAGE, nh, nkv, hd, 0, st)
    got = out.view(-1, nh, hd)
    assert st.item() == BAD_INDEX and (got[:64] == 0)[:, 0].all() and torch.isnan(got[70, 1]).all() and (got[:10] == 0).all() and (got[11:64] == 0).all()
    got[[10, 70], 1] = 0
    assert torch.isfinite(got).all()


def test_prefill_tiles_that_are_none():
    for hd in (128, 192):
        nh, nkv, news, pasts = 2, 1, [150, 140], [100, 30]
        table, k, v, exps, q, starts, tile_seq, tile_first = prefill_inputs(nh, nkv, hd, news, pasts, 8)
        out, st = torch.empty_like(q), status()
        ops.attn_prefill_kv8(q, k, v, exps, out, tile_seq, tile_first, ints(starts), ints(pasts), table, PAGE, nh, nkv, hd, 0, st)
        got = torch.full_like(q, 7)
        bad_seq, bad_first = torch.cat((tile_seq, ints([2, -1, 0]))), torch.cat((tile_first, ints([0, 0, -128])))
        ops.attn_prefill_kv8(q, k, v, exps, got, bad_seq, bad_first, ints(starts), ints(pasts), table, PAGE, nh, nkv, hd, 0, st)
        assert st.item() == BAD_INDEX and torch.equal(got, out)
        # positions that the table does not have: the sequence is left out, the other is not
        got.fill_(7)
        st.zero_()
        ops.attn_prefill_kv8(q, k, v, exps, got, tile_seq, tile_first, ints(starts), ints([64 * table.shape[1], 30]), table, PAGE, nh, nkv, hd, 0, st)
        assert st.item() == BAD_INDEX and torch.equal(got[150:], out[150:]) and (got[:128] == 7).all()


@pytest.mark.parametrize("hd", [64, 128, 192])
@pytest.mark.parametrize("first", [5, 64, 129, 384, 2 ** 31 - 1])
def test_prefill_tiles_between_the_tiles(hd, first):
    """A tile that is none of its sequence's is left out, the others are as without it."""
    nh, nkv, news, pasts = 2, 1, [300, 140], [100, 30]
    table, k, v, exps, q, starts, tile_seq, tile_first = prefill_inputs(nh, nkv, hd, news, pasts, 8)
    out, got, st = torch.empty_like(q), torch.full_like(q, 7), status()
    ops.attn_prefill_kv8(q, k, v, exps, out, tile_seq, tile_first, ints(starts), ints(pasts), table, PAGE, nh, nkv, hd, 0, st)
    assert st.item() == 0
    ops.attn_prefill_kv8(q, k, v, exps, got, torch.cat((ints([0]), tile_seq)), torch.cat((ints([first]), tile_first)), ints(starts), ints(pasts), table, PAGE,
                         nh, nkv, hd, 0, st)
    assert st.item() == BAD_INDEX and torch.equal(got, out)


@pytest.mark.parametrize("hd", [64, 128, 192])
@pytest.mark.parametrize("starts", [[0, 150, 291], [0, 150, 2 ** 31 - 1], [0, -5, 140], [-20, 150, 290]])
def test_prefill_rows_that_are_none(hd, starts):
    """Sequences whose rows the queries do not have are left out."""
    nh, nkv, news, pasts = 2, 1, [150, 140], [100, 30]
    table, k, v, exps, q, good, tile_seq, tile_first = prefill_inputs(nh, nkv, hd, news, pasts, 8)
    out, got, st = torch.empty_like(q), torch.full_like(q, 7), status()
    ops.attn_prefill_kv8(q, k, v, exps, out, tile_seq, tile_first, ints(good), ints(pasts), table, PAGE, nh, nkv, hd, 0, st)
    assert st.item() == 0
    ops.attn_prefill_kv8(q, k, v, exps, got, tile_seq, tile_first, ints(starts), ints(pasts), table, PAGE, nh, nkv, hd, 0, st)
    assert st.item() == BAD_INDEX
    for i in range(2):
        fine = 0 <= starts[i] < starts[i + 1] <= 290
        rows = slice(good[i], good[i + 1])
        assert torch.equal(got[rows], out[rows] if fine else torch.full_like(out[rows], 7))


@pytest.mark.parametrize("hd", [64, 96, 128, 192])
@pytest.mark.parametrize("news", [[150, 140], [14, 12]])
@pytest.mark.parametrize("end", ["one more", 2 ** 31 - 1, -2 ** 31, -1, 3])
def test_prefill_of_a_sequence_that_ends_nowhere(hd, news, end):
    """The second sequence's end lies behind the queries or ahead of its start, also where their difference is no 32-bit number, and
    also in calls that the streaming kernel has to itself (at most 32 rows): it is left out and the status says so."""
    nh, nkv, pasts = 2, 1, [100, 30]
    table, k, v, exps, q, good, tile_seq, tile_first = prefill_inputs(nh, nkv, hd, news, pasts, 8)
    out, got, st = torch.empty_like(q), torch.full_like(q, 7), status()
    ops.attn_prefill_kv8(q, k, v, exps, out, tile_seq, tile_first, ints(good), ints(pasts), table, PAGE, nh, nkv, hd, 0, st)
    assert st.item() == 0
    bad = [*good[:2], good[2] + 1 if end == "one more" else end]
    ops.attn_prefill_kv8(q, k, v, exps, got, tile_seq, tile_first, ints(bad), ints(pasts), table, PAGE, nh, nkv, hd, 0, st)
    assert st.item() == BAD_INDEX
    assert torch.equal(got[:good[1]], out[:good[1]]) and (got[good[1]:] == 7).all()


def test_prefill_bad_tiles_among_sequences_of_few_tokens():
    """Both kernels that share such a call leave out what is none, and each writes the rows of its own sequences alone."""
    nh, nkv, hd, news, pasts = 6, 2, 128, [130, 5, 40, 17, 3], [64, 700, 0, 300, 1]
    table, k, v, exps, q, starts, tile_seq, tile_first = prefill_inputs(nh, nkv, hd, news, pasts, 8)
    out, got, st = torch.empty_like(q), torch.full_like(q, 7), status()
    ops.attn_prefill_kv8(q, k, v, exps, out, tile_seq, tile_first, ints(starts), ints(pasts), table, PAGE, nh, nkv, hd, 0, st)
    assert st.item() == 0
    check_prefill(out, q, k, v, exps, table, starts, pasts, nh, hd, 0)
    for seqs, firsts in (([5], [0]), ([-1], [0]), ([1], [128]), ([0], [256]), ([4], [3])):
        st.zero_(), got.fill_(7)
        ops.attn_prefill_kv8(q, k, v, exps, got, torch.cat((ints(seqs), tile_seq)), torch.cat((ints(firsts), tile_first)), ints(starts), ints(pasts), table,
                             PAGE, nh, nkv, hd, 0, st)
        assert st.item() == BAD_INDEX and torch.equal(got, out)
    # two sequences' pasts reach beyond the page table
    st.zero_(), got.fill_(7)
    far = list(pasts)
    far[0] = far[3] = 64 * table.shape[1]
    ops.attn_prefill_kv8(q, k, v, exps, got, tile_seq, tile_first, ints(starts), ints(far), table, PAGE, nh, nkv, hd, 0, st)
    assert st.item() == BAD_INDEX
    for i in range(5):
        rows = slice(starts[i], starts[i + 1])
        assert torch.equal(got[rows], torch.full_like(out[rows], 7) if i in (0, 3) else out[rows])


@pytest.mark.parametrize("nh,hd", [(1, 64), (3, 128)])
def test_prefill_of_more_tiles_than_a_launch_lists(nh, hd):
    """5,000 sequences of one token: a row sees its own position alone, so the result is its value."""
    n = 5000
    k, v, exps = pools(n, 1, hd, 4)
    q = torch.randn((n, nh * hd), generator=gen(1), device="cuda").to(torch.bfloat16)
    order = torch.randperm(n, generator=torch.Generator().manual_seed(1)).to(torch.int32).cuda()
    out, st, seq = torch.full_like(q, math.nan), status(), torch.arange(n, dtype=torch.int32, device="cuda")
    ops.attn_prefill_kv8(q, k, v, exps, out, seq, ints([0] * n), torch.arange(n + 1, dtype=torch.int32, device="cuda"), ints([0] * n), order[:, None].contiguous(),
                         PAGE, nh, 1, hd, 0, st)
    want = plain.stored(v[order.long(), 0, 0], exps[order.long(), 0, 1, 0])
    assert st.item() == 0
    assert torch.equal(out.view(n, nh, hd).double(), want[:, None].expand(n, nh, hd))


def test_prefill_of_two_tiles_that_different_launches_list():
    """The second of a sequence's two tiles heads a list of 4,098, the first ends it."""
    nh, nkv, hd = 2, 1, 128
    news = [200] + [1] * 4096
    pasts = [0] * len(news)
    table, k, v, exps, q, starts, _, _ = prefill_inputs(nh, nkv, hd, news, pasts, 9)
    tile_seq, tile_first = ints([0, *range(1, 4097), 0]), ints([128, *[0] * 4096, 0])
    out, st = torch.full_like(q, math.nan), status()
    ops.attn_prefill_kv8(q, k, v, exps, out, tile_seq, tile_first, ints(starts), ints(pasts), table, PAGE, nh, nkv, hd, 0, st)
    assert st.item() == 0 and torch.isfinite(out).all()
    check_prefill(out[:200], q, k, v, exps, table, starts[:2], pasts[:1], nh, hd, 0)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_windows_beyond_all_positions(hd):
    """A window that reaches past the first position hides nothing, whatever its size."""
    nh, nkv, news, pasts = 2, 1, [140], [100]
    table, k, v, exps, q, starts, tile_seq, tile_first = prefill_inputs(nh, nkv, hd, news, pasts, 6)
    outs, ones, st, ws = [], [], status(), Workspace(q.device)
    for window in (None, 240, 2 ** 31 - 1, 2 ** 31, 2 ** 32 + 5):
        outs.append(torch.empty_like(q))
        ops.attn_prefill_kv8(q, k, v, exps, outs[-1], tile_seq, tile_first, ints(starts), ints(pasts), table, PAGE, nh, nkv, hd, window, st)
        ones.append(torch.empty_like(q[:1]))
        ops.attn_decode_kv8(q[-1:], k, v, exps, ones[-1], ws, ints([0]), ints([239]), table, PAGE, nh, nkv, hd, window, st)
    assert st.item() == 0 and all(torch.equal(outs[0], x) for x in outs) and all(torch.equal(ones[0], x) for x in ones)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_queries_that_are_no_numbers(hd, value):
    """A row whose query holds an infinity or a NaN is NaN, be its scores all the lowest or not; the others are not touched."""
    nh, nkv, news, pasts = 2, 1, [300], [40]
    table, k, v, exps, q, starts, tile_seq, tile_first = prefill_inputs(nh, nkv, hd, news, pasts, 6)
    k = k.view(torch.uint8).clone()
    k[..., 5] = 0x38                                       # 1: the query's infinity is every score's
    k = k.view(E4M3)
    rows, st = torch.tensor([0, 130, 299], device="cuda"), status()
    want, got, bad = torch.empty_like(q), torch.empty_like(q), q.clone()
    bad.view(-1, nh, hd)[rows, 1, 5] = value
    for qq, out in ((q, want), (bad, got)):
        ops.attn_prefill_kv8(qq, k, v, exps, out, tile_seq, tile_first, ints(starts), ints(pasts), table, PAGE, nh, nkv, hd, 0, st)
    hit = torch.zeros((300, nh), dtype=torch.bool, device="cuda")
    hit[rows, 1] = True
    assert torch.isnan(got.view(-1, nh, hd)[hit]).all() and torch.equal(got.view(-1, nh, hd)[~hit], want.view(-1, nh, hd)[~hit])
    one, ws = torch.empty_like(q[rows]), Workspace(q.device)
    ops.attn_decode_kv8(bad[rows], k, v, exps, one, ws, ints([0, 0, 0]), ints([40, 170, 339]), table, PAGE, nh, nkv, hd, 0, st)
    assert st.item() == 0 and torch.isnan(one.view(3, nh, hd)[:, 1]).all() and torch.isfinite(one.view(3, nh, hd)[:, 0]).all()


def scores_of_one_channel(hd, length, amplitude, best, seed):
    """Keys whose scores are amplitude / sqrt(hd) times 1 or 2: the largest are those of ``best`` (None: all the same).  (table, k, v, exps, query
    row of one head, the values in 64 bits)."""
    table, total = tables([length], 3)
    k, v, exps = pools(total, 1, hd, seed)
    k.view(torch.uint8).zero_()
    k.view(torch.uint8)[..., 0] = 0x40 if best is None or amplitude < 0 else 0x38          # 2 and 1
    exps[:, :, 0] = 127
    if best is not None:
        k.view(torch.uint8)[table[0, best // PAGE].long(), 0, best % PAGE, 0] = 0x38 if amplitude < 0 else 0x40
    q = torch.zeros(hd, device="cuda", dtype=torch.bfloat16)
    q[0] = amplitude
    return table, k, v, exps, q, sequence_rows(v, exps, 1, table[0, :(length + PAGE - 1) // PAGE].long(), length)[0]


@pytest.mark.parametrize("nh,hd", [(1, 64), (3, 128), (12, 128), (2, 192), (1, 256)])
@pytest.mark.parametrize("amplitude", [1e3, 1e7, 3e8, 1e10, 1e15, 1e30, 3e38, -1e7, -1e10, -1e30])
def test_scores_of_any_size(nh, hd, amplitude):
    """The value of the one key whose score is far above the others, or the mean where all are the same, be the scores themselves beyond
    what a value's exponent can be added to."""
    length, new = 700, 30
    for best in (5, 300, 660, None):
        table, k, v, exps, row, values = scores_of_one_channel(hd, length, amplitude, best, 5)
        q = row.repeat(new, nh)
        one, st = torch.full_like(q, math.nan), status()
        pos = torch.arange(length - new, length, dtype=torch.int32, device="cuda")
        ops.attn_decode_kv8(q, k, v, exps, one, Workspace(q.device), ints([0] * new), pos, table, PAGE, nh, 1, hd, 0, st)
        outs = [one]
        if hd > 64:                                       # runs of few tokens and wide heads: the streaming kernel as well
            outs.append(torch.full_like(q, math.nan))
            ops.attn_prefill_kv8(q, k, v, exps, outs[-1], ints([0]), ints([0]), ints([0, new]), ints([length - new]), table, PAGE, nh, 1, hd, 0, st)
        assert st.item() == 0
        want = torch.stack([values[best] if best is not None else values[:p + 1].mean(0) for p in pos.tolist()])[:, None]
        spread = torch.stack([values[best].abs() if best is not None else values[:p + 1].abs().mean(0) for p in pos.tolist()])[:, None]
        for out in outs:
            off = (out.double().view(new, nh, hd) - want).abs()
            # the result's rounding; weights are halfs (2^-11), exp2 and sums are 32-bit
            assert torch.all(off <= 2.0 ** -8 * want.abs() + 2.0 ** -10 * spread + 1e-30), (best, float(off.max()))


@pytest.mark.parametrize("nh,hd,new", [(1, 64, 300), (3, 128, 140), (100, 64, 400), (2, 104, 40)])
@pytest.mark.parametrize("amplitude", [1e3, 1e7, 3e8, 2e9, -1e7, -2e9])
def test_scores_of_prompts_below_their_bound(nh, hd, new, amplitude):
    """The same of the tensor-memory kernel, for scores of up to 2^29 in units of log2."""
    length = 700
    for best in (5, 150, None):
        table, k, v, exps, row, values = scores_of_one_channel(hd, length, amplitude, best, 5)
        q, st = row.repeat(new, nh), status()
        out = torch.full_like(q, math.nan)
        firsts = list(range(0, new, 128))
        ops.attn_prefill_kv8(q, k, v, exps, out, ints([0] * len(firsts)), ints(firsts), ints([0, new]), ints([length - new]), table, PAGE, nh, 1, hd, 0, st)
        assert st.item() == 0
        pos = range(length - new, length)
        want = torch.stack([values[best] if best is not None else values[:p + 1].mean(0) for p in pos])[:, None]
        spread = torch.stack([values[best].abs() if best is not None else values[:p + 1].abs().mean(0) for p in pos])[:, None]
        off = (out.double().view(new, nh, hd) - want).abs()
        # the result's rounding; weights are bfloat16 (2^-8), exp2 and sums are 32-bit
        assert torch.all(off <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -20) * (1 + 2.0 ** -8) * spread + 1e-30), (best, float(off.max()))


# ------------------------------------------------------------------------------------------------------- together
def test_pools_past_32_bits_of_bytes():
    """Pages whose codes lie more than 2^31 bytes into the pool."""
    nh, nkv, hd, pages = 4, 4, 256, 34000
    k, v = (torch.empty((pages, nkv, PAGE, hd), dtype=E4M3, device="cuda") for _ in range(2))
    exps = torch.zeros((pages, nkv, 2, PAGE), dtype=torch.uint8, device="cuda")
    assert k.numel() > 1 << 31
    for hd_now in (256, 128):
        kk, vv = k.view(-1, nkv, PAGE, hd_now)[:2 * pages if hd_now == 128 else pages], v.view(-1, nkv, PAGE, hd_now)
        ee = exps if hd_now == 256 else torch.zeros((2 * pages, nkv, 2, PAGE), dtype=torch.uint8, device="cuda")
        last = kk.shape[0]
        table = ints([[last - 1, last - 3, last - 2, -1]])
        n, length = 150, 150
        qkv = torch.randn((n, 3 * nh * hd_now), generator=gen(2), device="cuda")
        q, st = torch.empty((n, nh * hd_now), dtype=torch.bfloat16, device="cuda"), status()
        seq, pos = ints([0] * n), torch.arange(n, dtype=torch.int32, device="cuda")
        ops.kv8_rope_append(qkv, None, seq, pos, None, None, 0, q, kk, vv, ee, table, PAGE, nh, nkv, hd_now, True, st)
        out, one = torch.empty_like(q), torch.empty_like(q[:1])
        ops.attn_prefill_kv8(q, kk, vv, ee, out, ints([0, 0]), ints([128, 0]), ints([0, n]), ints([0]), table, PAGE, nh, nkv, hd_now, 0, st)
        ops.attn_decode_kv8(q[-1:], kk, vv, ee, one, Workspace(q.device), ints([0]), ints([n - 1]), table, PAGE, nh, nkv, hd_now, 0, st)
        assert st.item() == 0
        check_prefill(out, q, kk, vv, ee, table, [0, n], [0], nh, hd_now, 0)
        check_decode(one, q[-1:], kk, vv, ee, table, [length], nh, hd_now, 0)


def test_calls_on_two_streams_with_a_workspace_each():
    """Decode and prefill of two steps at once: nothing is shared but the pools."""
    nh, nkv, hd, lengths = 8, 2, 128, [3000, 700, 1500]
    table, k, v, exps, q, seq, pos = decode_inputs(nh, nkv, hd, lengths, 4)
    want, st = torch.empty_like(q), status()
    ops.attn_decode_kv8(q, k, v, exps, want, Workspace(q.device), seq, pos, table, PAGE, nh, nkv, hd, 0, st)
    torch.cuda.synchronize()
    streams, outs, spaces = [torch.cuda.Stream() for _ in range(2)], [torch.empty_like(q) for _ in range(2)], [Workspace(q.device) for _ in range(2)]
    for stream, ws in zip(streams, spaces):               # the scratch is made on the stream that uses it
        with torch.cuda.stream(stream):
            ops.attn_decode_kv8(q, k, v, exps, outs[0], ws, seq, pos, table, PAGE, nh, nkv, hd, 0, st)
    torch.cuda.synchronize()
    for _ in range(20):
        for stream, out, ws in zip(streams, outs, spaces):
            with torch.cuda.stream(stream):
                ops.attn_decode_kv8(q, k, v, exps, out, ws, seq, pos, table, PAGE, nh, nkv, hd, 0, st)
    torch.cuda.synchronize()
    assert st.item() == 0 and torch.equal(outs[0], want) and torch.equal(outs[1], want)


@pytest.mark.parametrize("nh,nkv,hd,news,pasts", [(8, 2, 128, [700, 300, 20], [300, 0, 900]), (32, 4, 64, [1300, 129], [0, 333]), (3, 3, 192, [200, 7], [90, 1000])])
def test_prefill_beside_other_calls_on_streams_of_their_own(nh, nkv, hd, news, pasts):
    """Prompts on two streams and decode on a third, over the same pools at once: the bits of calls behind one another."""
    table, k, v, exps, q, starts, tile_seq, tile_first = prefill_inputs(nh, nkv, hd, news, pasts, 14)
    st, n = status(), len(news)
    seq, pos = torch.arange(n, dtype=torch.int32, device="cuda"), ints([a + b - 1 for a, b in zip(pasts, news)])
    rows = torch.tensor([b - 1 for b in starts[1:]], device="cuda")
    one_q = q[rows].contiguous()
    args = (tile_seq, tile_first, ints(starts), ints(pasts), table, PAGE, nh, nkv, hd, 0, st)
    spaces = [Workspace(q.device) for _ in range(3)]
    calls = [lambda out, ws: ops.attn_prefill_kv8(q, k, v, exps, out, *args), lambda out, ws: ops.attn_prefill_kv8(q, k, v, exps, out, *args),
             lambda out, ws: ops.attn_decode_kv8(one_q, k, v, exps, out, ws, seq, pos, table, PAGE, nh, nkv, hd, 0, st)]
    streams, outs = [torch.cuda.Stream() for _ in calls], [torch.empty_like(q), torch.empty_like(q), torch.empty_like(one_q)]
    wants = [torch.empty_like(x) for x in outs]
    torch.cuda.synchronize()
    for call, stream, want, ws in zip(calls, streams, wants, spaces):
        with torch.cuda.stream(stream):
            call(want, ws)
        torch.cuda.synchronize()
    for _ in range(20):
        for call, stream, out, ws in zip(calls, streams, outs, spaces):
            with torch.cuda.stream(stream):
                call(out, ws)
    torch.cuda.synchronize()
    assert st.item() == 0 and all(torch.equal(a, b) for a, b in zip(outs, wants))
    check_prefill(wants[0], q, k, v, exps, table, starts, pasts, nh, hd, 0)


def test_a_first_call_is_not_captured():
    """The counters' zeros would be the graph's; refused, and the same workspace serves an eager call afterwards."""
    nh, nkv, hd, lengths = 8, 2, 128, [3000, 700]
    table, k, v, exps, q, seq, pos = decode_inputs(nh, nkv, hd, lengths, 4)
    out, st, ws, graph = torch.empty_like(q), status(), Workspace(q.device), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with pytest.raises(Backend, match="captured"), torch.cuda.graph(graph):
        ops.attn_decode_kv8(q, k, v, exps, out, ws, seq, pos, table, PAGE, nh, nkv, hd, 0, st)
    del graph
    ops.attn_decode_kv8(q, k, v, exps, out, ws, seq, pos, table, PAGE, nh, nkv, hd, 0, st)
    assert st.item() == 0
    check_decode(out, q, k, v, exps, table, lengths, nh, hd, 0)


def test_append_then_attend_is_a_captured_step():
    """A step as it is used, append then decode, on a stream of its own and replayed from a graph over changing inputs."""
    nh, nkv, hd, lengths = 8, 2, 128, [130, 700]
    n, width = 2, (nh + 2 * nkv) * hd
    table, total = tables([length + 8 for length in lengths], 3)
    k, v, exps = pools(total, nkv, hd, 2)
    angle = torch.arange(800, device="cuda")[:, None] * 1e4 ** (-torch.arange(64, device="cuda") / 64)
    cos, sin = angle.cos().contiguous(), angle.sin().contiguous()
    qkv, q = torch.empty((n, width), device="cuda"), torch.empty((n, nh * hd), dtype=torch.bfloat16, device="cuda")
    out, st, ws, seq, pos = torch.empty_like(q), status(), Workspace(q.device), ints([0, 1]), ints([0, 0])

    def step():
        ops.kv8_rope_append(qkv, None, seq, pos, cos, sin, hd, q, k, v, exps, table, PAGE, nh, nkv, hd, True, st)
        ops.attn_decode_kv8(q, k, v, exps, out, ws, seq, pos, table, PAGE, nh, nkv, hd, 0, st)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        pos.copy_(ints([length - 1 for length in lengths]))
        qkv.normal_()
        step()
        graph = torch.cuda.CUDAGraph()
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            step()
        for t in range(4):
            now = [length + t for length in lengths]
            pos.copy_(ints([length - 1 for length in now]))
            qkv.normal_()
            graph.replay()
            side.synchronize()
            assert st.item() == 0
            check_decode(out, q, k, v, exps, table, now, nh, hd, 0)


@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 128), (4, 4, 64), (2, 1, 192)])
def test_a_captured_prompt_over_changing_inputs(nh, nkv, hd):
    """Append and attention of many tokens in a graph, replayed over other numbers, pages, lengths and cached positions of as many rows."""
    n, width, longest = 260, (nh + 2 * nkv) * hd, 700
    k, v, exps = pools(40, nkv, hd, 2)
    angle = torch.arange(longest, device="cuda")[:, None] * 1e4 ** (-torch.arange(hd // 2, device="cuda") / (hd // 2))
    cos, sin = angle.cos().contiguous(), angle.sin().contiguous()
    qkv, q = torch.empty((n, width), device="cuda"), torch.empty((n, nh * hd), dtype=torch.bfloat16, device="cuda")
    out, st = torch.empty_like(q), status()
    # three tiles either way: 200 and 60 new tokens, or 20 and 240
    lists = {name: torch.zeros(size, dtype=torch.int32, device="cuda") for name, size in
             (("seq", n), ("pos", n), ("tile_seq", 3), ("tile_first", 3), ("start", 3), ("past", 2))}
    table = torch.zeros((2, longest // PAGE + 1), dtype=torch.int32, device="cuda")

    def fill(news, pasts, seed):
        starts = [0, news[0], n]
        for name, what in (("seq", [i for i, t in enumerate(news) for _ in range(t)]), ("pos", [p + j for p, t in zip(pasts, news) for j in range(t)]),
                           ("tile_seq", [i for i, t in enumerate(news) for _ in range(0, t, 128)]),
                           ("tile_first", [f for t in news for f in range(0, t, 128)]), ("start", starts), ("past", pasts)):
            lists[name].copy_(ints(what))
        table.copy_(torch.randperm(40, generator=torch.Generator().manual_seed(seed))[:table.numel()].to(torch.int32).view_as(table))
        qkv.normal_()
        return starts

    def step():
        ops.kv8_rope_append(qkv, None, lists["seq"], lists["pos"], cos, sin, hd, q, k, v, exps, table, PAGE, nh, nkv, hd, True, st)
        ops.attn_prefill_kv8(q, k, v, exps, out, lists["tile_seq"], lists["tile_first"], lists["start"], lists["past"], table, PAGE, nh, nkv, hd, 0, st)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fill([200, 60], [0, 100], 1)
        step()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
        for i, (news, pasts) in enumerate([([200, 60], [300, 5]), ([20, 240], [500, 0]), ([240, 20], [1, 640])]):
            starts = fill(news, pasts, i)
            out.fill_(math.nan)
            graph.replay()
            side.synchronize()
            assert st.item() == 0
            check_prefill(out, q, k, v, exps, table, starts, pasts, nh, hd, 0)
    del graph


@pytest.mark.parametrize("nh,nkv,hd,news,pasts", [(2, 1, 128, [150, 20], [0, 70]), (16, 16, 64, [1500, 300], [0, 5]), (2, 2, 192, [40, 17], [9, 0]), (2, 1, 96, [9, 2], [0, 70])])
def test_rows_behind_the_last_sequence_and_tiles_listed_twice(nh, nkv, hd, news, pasts):
    table, k, v, exps, q, starts, tile_seq, tile_first = prefill_inputs(nh, nkv, hd, news, pasts, 3)
    want, st = torch.empty_like(q), status()
    ops.attn_prefill_kv8(q, k, v, exps, want, tile_seq, tile_first, ints(starts), ints(pasts), table, PAGE, nh, nkv, hd, 0, st)
    padded = torch.cat((q, torch.full_like(q[:50], math.nan)))
    out = torch.full_like(padded, 7)
    ops.attn_prefill_kv8(padded, k, v, exps, out, torch.cat((tile_seq, tile_seq)), torch.cat((tile_first, tile_first)), ints(starts), ints(pasts), table, PAGE,
                         nh, nkv, hd, 0, st)
    assert st.item() == 0 and (out[starts[-1]:] == 7).all()
    check_prefill(out, q, k, v, exps, table, starts, pasts, nh, hd, 0)
    check_prefill(want, q, k, v, exps, table, starts, pasts, nh, hd, 0)


@pytest.mark.parametrize("nh,nkv,hd", [(2, 1, 8), (200, 1, 64), (130, 2, 96), (1, 1, 136)])
def test_the_smallest_heads_and_the_most_of_them(nh, nkv, hd):
    news, pasts = [140, 3], [10, 129]
    table, k, v, exps, q, starts, tile_seq, tile_first = prefill_inputs(nh, nkv, hd, news, pasts, 12)
    out, one, st = torch.full_like(q, math.nan), torch.full_like(q, math.nan), status()
    ops.attn_prefill_kv8(q, k, v, exps, out, tile_seq, tile_first, ints(starts), ints(pasts), table, PAGE, nh, nkv, hd, 0, st)
    seq = ints([i for i, t in enumerate(news) for _ in range(t)])
    pos = ints([past + j for past, t in zip(pasts, news) for j in range(t)])
    ops.attn_decode_kv8(q, k, v, exps, one, Workspace(q.device), seq, pos, table, PAGE, nh, nkv, hd, 0, st)
    assert st.item() == 0
    check_prefill(out, q, k, v, exps, table, starts, pasts, nh, hd, 0)
    check_prefill(one, q, k, v, exps, table, starts, pasts, nh, hd, 0)


def test_prefill_and_decode_agree():
    """The last row of a run sees what a decode step at its place sees."""
    for hd, weight in ((128, 2.0 ** -8), (192, 2.0 ** -11)):
        nh, nkv, news, pasts = 6, 2, [200, 129], [0, 300]
        table, k, v, exps, q, starts, tile_seq, tile_first = prefill_inputs(nh, nkv, hd, news, pasts, 2)
        out, st = torch.empty_like(q), status()
        ops.attn_prefill_kv8(q, k, v, exps, out, tile_seq, tile_first, ints(starts), ints(pasts), table, PAGE, nh, nkv, hd, 0, st)
        rows = torch.tensor([starts[1] - 1, starts[2] - 1], device="cuda")
        one = torch.empty((2, nh * hd), dtype=torch.bfloat16, device="cuda")
        ops.attn_decode_kv8(q[rows], k, v, exps, one, Workspace(q.device), ints([0, 1]), ints([199, 428]), table, PAGE, nh, nkv, hd, 0, st)
        spread = torch.nan_to_num(plain.stored(v, exps[:, :, 1])).abs().max()
        assert (one.double() - out[rows].double()).abs().max() <= (2 * 2.0 ** -8 + weight + 2.0 ** -11 + 1e-3) * spread
