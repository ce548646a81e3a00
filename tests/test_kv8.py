"""The 8-bit cache without a GPU: the plain implementation that the kernels are compared with, and what the entry points refuse."""
import math

import pytest
import torch

import plain_kv8 as plain
from esp_b200.csrc import ops
from esp_b200.errors import Backend

E4M3 = torch.float8_e4m3fn


def test_plain_e4m3_is_the_type_s_own_rounding():
    grid = plain.e4m3_values()
    assert grid[-1] == 448 and grid[1] == 2.0 ** -9 and len(grid) == 127
    x = torch.cat((grid, -grid, (grid[1:] + grid[:-1]) / 2, torch.randn(20000, dtype=torch.float64) * torch.exp(3 * torch.randn(20000, dtype=torch.float64))))
    x = x.clamp(-448, 448).float()
    assert torch.equal(plain.round_e4m3(x.double()), x.to(E4M3).double())


def test_plain_exponents():
    amax = torch.tensor([0.0, 448.0, 448.0 * (1 + 2.0 ** -23), 224.0, 224.01, 1e-300, 448 * 2.0 ** -100, 449 * 2.0 ** -100, 448 * 2.0 ** 100], dtype=torch.float64)
    assert plain.row_exponent(amax).tolist() == [-100, 0, 1, -1, 0, -100, -100, -99, 100]
    codes, e = plain.quantize(torch.tensor([[1.0, math.inf], [math.nan, 0.0], [2.0 ** 110, 1.0], [3.0, -1.0]], dtype=torch.float64))
    assert torch.isnan(e).tolist() == [True, True, True, False] and not codes[:3].any()
    assert (codes[3] * 2.0 ** e[3]).tolist() == [3.0, -1.0]


def args(nh=4, nkv=2, hd=64, n=3, pages=5, page=64):
    return dict(q=torch.zeros((n, nh * hd), dtype=torch.bfloat16), k=torch.zeros((pages, nkv, page, hd), dtype=E4M3),
                v=torch.zeros((pages, nkv, page, hd), dtype=E4M3), exps=torch.zeros((pages, nkv, 2, page), dtype=torch.uint8),
                out=torch.zeros((n, nh * hd), dtype=torch.bfloat16), table=torch.zeros((2, 4), dtype=torch.int32),
                seq=torch.zeros(n, dtype=torch.int32), pos=torch.zeros(n, dtype=torch.int32), page=page, nh=nh, nkv=nkv, hd=hd, window=0)


def decode(a):
    ops.attn_decode_kv8(a["q"], a["k"], a["v"], a["exps"], a["out"], None, a["seq"], a["pos"], a["table"], a["page"], a["nh"], a["nkv"], a["hd"],
                        a["window"], torch.zeros(1, dtype=torch.int32))


def prefill(a):
    ops.attn_prefill_kv8(a["q"], a["k"], a["v"], a["exps"], a["out"], a["seq"], a["seq"], a["pos"], a["pos"], a["table"], a["page"], a["nh"], a["nkv"],
                         a["hd"], a["window"], torch.zeros(1, dtype=torch.int32))


WRONG = [
    ({"nkv": 3}, "do not divide"),
    ({"hd": 60}, "multiples of 8"),
    ({"hd": 264}, "multiples of 8"),
    ({"page": 32}, "pages of"),
    ({"q": torch.zeros((3, 100), dtype=torch.bfloat16), "out": torch.zeros((3, 100), dtype=torch.bfloat16)}, "queries of shape"),
    ({"k": torch.zeros((5, 2, 64, 32), dtype=E4M3)}, "pools of shape"),
    ({"v": torch.zeros((4, 2, 64, 64), dtype=E4M3)}, "pools of shape"),
    ({"exps": torch.zeros((5, 2, 64, 2), dtype=torch.uint8)}, "exponents of shape"),
    ({"table": torch.zeros(8, dtype=torch.int32)}, "page table"),
    ({"out": torch.zeros((2, 256), dtype=torch.bfloat16)}, "for the results"),
    ({"window": -1}, "window"),
    ({"k": torch.zeros(5 * 2 * 64 * 64 + 1, dtype=torch.uint8)[1:].view(E4M3).view(5, 2, 64, 64)}, "multiple of 16"),
    ({}, "no CPU path"),
]


@pytest.mark.parametrize("call", [decode, prefill])
@pytest.mark.parametrize("change,why", WRONG)
def test_attention_refuses(call, change, why):
    with pytest.raises(Backend, match=why):
        call({**args(), **change})


def test_decode_refuses_short_lists():
    a = args()
    for name in ("seq", "pos"):
        with pytest.raises(Backend, match="tok_" + name):
            decode({**a, name: torch.zeros(2, dtype=torch.int32)})
    with pytest.raises(Backend, match="seq_start"):
        prefill({**a, "pos": torch.zeros(2, dtype=torch.int32)})


def test_attention_refuses_tables_whose_positions_are_no_32_bit_numbers():
    """2^25 pages hold 2^31 positions; 1,024 rows of 2^22 pages may see 2^38 keys."""
    a = {**args(), "table": torch.zeros((1, 1 << 25), dtype=torch.int32)}
    for call in (decode, prefill):
        with pytest.raises(Backend, match="pages a sequence"):
            call(a)
    n = 1100
    a = {**args(n=n), "table": torch.zeros((1, 1 << 22), dtype=torch.int32), "seq": torch.zeros(n, dtype=torch.int32), "pos": torch.zeros(n, dtype=torch.int32)}
    with pytest.raises(Backend, match="too many for a launch"):
        decode(a)
    for table, rows in (((1 << 25) - 1, 3), ((1 << 22) - 4, n)):
        a = {**args(n=rows), "table": torch.zeros((1, table), dtype=torch.int32), "seq": torch.zeros(rows, dtype=torch.int32),
             "pos": torch.zeros(rows, dtype=torch.int32)}
        with pytest.raises(Backend, match="no CPU path"):
            decode(a)


def append(**change):
    nh, nkv, hd, n = 4, 2, 64, 3
    a = dict(qkv=torch.zeros((n, (nh + 2 * nkv) * hd)), bias=None, seq=torch.zeros(n, dtype=torch.int32), pos=torch.zeros(n, dtype=torch.int32),
             cos=torch.zeros((9, 32)), sin=torch.zeros((9, 32)), rot=64, q=torch.zeros((n, nh * hd), dtype=torch.bfloat16), write=True)
    b = args(nh, nkv, hd, n)
    a.update(k=b["k"], v=b["v"], exps=b["exps"])
    a.update(change)
    ops.kv8_rope_append(a["qkv"], a["bias"], a["seq"], a["pos"], a["cos"], a["sin"], a["rot"], a["q"], a["k"], a["v"], a["exps"], b["table"], 64, nh, nkv,
                        hd, a["write"], torch.zeros(1, dtype=torch.int32))


@pytest.mark.parametrize("change,why", [
    ({"qkv": torch.zeros((3, 500))}, "width"), ({"rot": 3}, "rotated"), ({"rot": 66}, "rotated"), ({"rot": 32}, "cosines"), ({"cos": None}, "cosines"),
    ({"sin": torch.zeros((8, 32))}, "cosines"), ({"k": None}, "no pools"), ({"q": torch.zeros((2, 256), dtype=torch.bfloat16)}, "rows for the queries"),
    ({"bias": torch.zeros(5)}, "bias"), ({"pos": torch.zeros(2, dtype=torch.int32)}, "tok_pos"), ({}, "no CPU path"),
    ({"write": False, "k": None}, "no CPU path"),
])
def test_append_refuses(change, why):
    with pytest.raises(Backend, match=why):
        append(**change)
