"""The engine, the entry point and the command line with keys and values in 8 bits."""
import json

import numpy as np
import pytest
import torch

import plain_kv8 as kv8
from esp_b200.cache import PAGE
from esp_b200.engine import Engine, StepEntry
from esp_b200.errors import InvalidRequest, Unsupported
from esp_b200.provider import DecoderProvider, GenerationRequest
from gpu_util import run_steps, steps_batches, steps_tail, steps_whole
from test_gpu_kv8_kernels import check_rows
from tiny import CASES, make_folder, random_ids

pytestmark = pytest.mark.gpu
LENGTHS = {"A": [100, 45, 128, 1], "B": [200, 40, 250, 65], "C": [150, 40, 160, 2]}


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    tmp = tmp_path_factory.mktemp("models")
    return {case: make_folder(tmp, case) for case in CASES}


@pytest.fixture(scope="module")
def engines(folders):
    made = {}

    def get(case, **kw):
        key = (case, tuple(sorted(kw.items())))
        if key not in made:
            made[key] = Engine.from_folder(folders[case], dtype="bfloat16", cache_dtype="float8_e4m3", **{"max_tokens": 2048, **kw})
        return made[key]
    return get


class Nothing:
    def take(self, *a):
        pass


def watch(engine, monkeypatch):
    """Compares every call of the attention with the definition: new rows of the pools with the projection's, the result with
    what the pools hold.  Returns the number of calls so far."""
    from esp_b200.parts.attention import Attention
    calls = [0]
    inner = Attention.attend

    def attend(self, q, o, ctx, layer):
        inner(self, q, o, ctx, layer)
        s, rt = self.spec, self.rt
        n = q.shape[0]
        nh, nkv, hd = s.num_heads, s.num_kv_heads, s.head_dim
        table = ctx.block_tables[layer.group].long()
        seq, pos = ctx.tok_seq.long(), ctx.tok_pos.long()
        qkv = rt.ws.get("attn_qkv", (n, self.qkv_width), torch.float32).double()
        x = (qkv if self.b_qkv is None else qkv + self.b_qkv.double()).view(n, nh + 2 * nkv, hd)
        turned = x.clone()
        turned[:, :nh + nkv] = kv8.rotate(x[:, :nh + nkv], self.position.cos.double()[pos], self.position.sin.double()[pos], hd)
        page, place = table[seq, pos // PAGE], pos % PAGE
        slack = 2.0 ** -20 * x.abs().amax()               # the rotation's roundings in 32-bit
        assert torch.all((q.view(n, nh, hd).double() - turned[:, :nh]).abs() <= 2.0 ** -8 * turned[:, :nh].abs() + slack)
        if layer.writes:
            for pool, which, lo in ((layer.k, 0, nh), (layer.v, 1, nh + nkv)):
                rows, e = kv8.stored(pool[page, :, place], layer.exps[page, :, which, place]), layer.exps[page, :, which, place].double() - 127
                half = torch.maximum(2.0 ** -4 * turned[:, lo:lo + nkv].abs(), torch.exp2(e - 10)[..., None])
                assert torch.all((rows - turned[:, lo:lo + nkv]).abs() <= half + slack)
        weight = 2.0 ** -8 if n > 128 and hd <= 128 else 2.0 ** -11
        starts, pasts, news = ctx.host["starts"], ctx.host["pasts"], ctx.host["news"]
        for i, (a, past, new) in enumerate(zip(starts, pasts, news)):
            length = past + new
            pages = table[i, :(length + PAGE - 1) // PAGE].clamp_min(0)
            kk, vv = (kv8.stored(p[pages], layer.exps[pages, :, w]).transpose(0, 1).flatten(1, 2)[:, :length] for p, w in ((layer.k, 0), (layer.v, 1)))
            qq = q[a:a + new].double().view(new, nh, hd)
            want, spread = kv8.attend(qq, torch.nan_to_num(kk), torch.nan_to_num(vv), torch.arange(past, length, device=q.device), s.window or 0)
            check_rows(o[a:a + new].double().view(new, nh, hd), want, spread, qq, kk, hd, weight)
        calls[0] += 1

    monkeypatch.setattr(Attention, "attend", attend)
    return calls


def requests_for(case):
    rng = np.random.default_rng(5)
    return {f"r{i}": random_ids(rng, n, CASES[case][0]["vocab_size"]) for i, n in enumerate(LENGTHS[case])}


@pytest.mark.parametrize("case", ["A", "B", "C"])
@pytest.mark.parametrize("cut", ["whole", "tail", "batches"])
def test_every_attention_call_is_the_definition(engines, monkeypatch, case, cut):
    eng = engines(case)
    reqs = requests_for(case)
    calls = watch(eng, monkeypatch)
    eng.use_graphs = False
    try:
        lens = {rid: max(1, len(t) - d) for (rid, t), d in zip(reqs.items(), [9, 5, 3, 0])}
        steps = {"whole": lambda: steps_whole(reqs), "tail": lambda: steps_tail(reqs, 6),
                 "batches": lambda: steps_batches(reqs, [["r0", "r1", "r3"], ["r2", "r1"]], lens)}[cut]()
        run_steps(eng, steps, Nothing())
    finally:
        eng.use_graphs = True
    assert calls[0] >= len(steps) * len(eng.plan.schedule)
    assert all(g.pool.available == g.pool.n for g in eng.cache.book.groups)


def test_sizes_of_the_cache_and_its_count(engines, folders):
    eng = engines("A")
    wide = Engine.from_folder(folders["A"], dtype="bfloat16", max_tokens=2048)
    s = eng.cache.layouts[0]
    layers = sum(len(m) for m in eng.cache.members)
    assert eng.cache.bytes_per_token() == layers * s.num_kv_heads * (2 * s.head_dim + 2)
    assert wide.cache.bytes_per_token() == layers * s.num_kv_heads * 4 * s.head_dim
    assert eng.memory_plan["cache_bytes"] == 2048 * eng.cache.bytes_per_token()
    held = sum(t.numel() for pools in (eng.cache.k_pools, eng.cache.v_pools, eng.cache.exp_pools) for t in pools)
    assert held == eng.memory_plan["cache_bytes"]
    before = eng.counters()["kv_bytes_read"]
    slot = eng.open()
    eng.step([StepEntry(slot, [1, 2, 3], [])])
    eng.close(slot)
    assert eng.counters()["kv_bytes_read"] - before == 3 * eng.cache.bytes_per_token()


def test_captured_steps_give_what_eager_steps_give(folders):
    """Greedy tokens and the logits' bits, replayed and eager; slots and pages used again in between."""
    rng = np.random.default_rng(1)
    prompts = [random_ids(rng, n, CASES["A"][0]["vocab_size"]) for n in (60, 3, 17)]
    outs, bits = [], []
    for graphs in (True, False):
        prov = DecoderProvider.load(folders["A"], cache_dtype="float8_e4m3", max_batch=3, max_tokens=3 * 128)
        prov.engine.use_graphs = graphs
        reqs = [GenerationRequest(prompt_ids=p, max_tokens=40) for p in prompts]
        outs.append([[g.token_ids for g in prov.generate(reqs)] for _ in range(2)])
        bits.append(prov.next_token_logits(prompts[0]))
        assert (prov.engine.graph_replays > 0) == graphs
        assert prov.engine.read_status() == 0
    assert outs[0] == outs[1] and outs[0][0] == outs[0][1]
    assert torch.equal(bits[0], bits[1])


def test_a_shared_cache_is_read_and_not_written(folders):
    from dataclasses import replace

    from esp_b200.config import config_from_json
    from esp_b200.config.plan import ScheduleEntry
    config = config_from_json(folders["A"])
    inner = config.plan

    def plan():
        p = inner()
        return replace(p, schedule=[ScheduleEntry(0, None), ScheduleEntry(0, 0), ScheduleEntry(1, None)])
    config.plan = plan
    from esp_b200.weights import FolderSource
    eng = Engine(config, lambda specs: FolderSource(folders["A"]), cache_dtype="float8_e4m3", max_tokens=512)
    assert eng.cache.layers[1].k is eng.cache.layers[0].k or eng.cache.layers[1].k.data_ptr() == eng.cache.layers[0].k.data_ptr()
    assert not eng.cache.layers[1].writes and eng.cache.layers[1].exps.data_ptr() == eng.cache.layers[0].exps.data_ptr()
    seen = []
    from esp_b200.csrc import ops
    real = ops.kv8_rope_append
    ops.kv8_rope_append = lambda *a: (seen.append(a[-2]), real(*a))[1]
    try:
        slot = eng.open()
        logits = eng.step([StepEntry(slot, [5, 6, 7], [2])])
        eng.close(slot)
    finally:
        ops.kv8_rope_append = real
    assert seen == [True, False, True] and torch.isfinite(logits).all() and eng.read_status() == 0


def test_refusals(folders):
    for dtype, cache in (("float32", "float8_e4m3"), ("bfloat16", "float8_e5m2"), ("bfloat16", "float32"), ("bfloat16", torch.float16)):
        with pytest.raises(InvalidRequest):
            Engine.from_folder(folders["A"], dtype=dtype, cache_dtype=cache, max_tokens=256)
    assert Engine.from_folder(folders["A"], dtype="bfloat16", cache_dtype="bfloat16", max_tokens=256).cache.exp_pools == [None]
    import galirax_cases
    import satavik_cases
    import vumedra_cases
    from esp_b200.config import config_from_dict
    for raw in (galirax_cases.CASES, satavik_cases.CASES, vumedra_cases.CASES):
        raw = next(iter(raw.values()))
        raw = raw[0] if isinstance(raw, tuple) else raw
        with pytest.raises(Unsupported, match="cache_dtype"):
            Engine.from_random(config_from_dict(raw), cache_dtype="float8_e4m3", max_tokens=256)


def test_command_line(folders, capsys):
    from esp_b200.cli import main
    out = []
    for extra in ([], ["--cache-dtype", "float8_e4m3"]):
        assert main(["generate", "--model", str(folders["A"]), "--prompt-ids", "5,17,3", "--max-tokens", "6", *extra]) == 0
        out.append(json.loads(capsys.readouterr().out.strip()))
    assert len(out[1]["token_ids"]) == 6 and out[1]["finish_reason"] == out[0]["finish_reason"]
    assert main(["generate", "--model", str(folders["A"]), "--prompt-ids", "5", "--dtype", "float32", "--cache-dtype", "float8_e4m3"]) == 1
    assert "8-bit cache" in capsys.readouterr().err


def test_heads_of_real_size_with_long_contexts(monkeypatch):
    """Heads of 128 as the large models have them: a prompt of many tokens, then a mixed step, then decode past several pages."""
    from esp_b200.config import config_from_dict
    raw = {**CASES["A"][0], "hidden_size": 256, "num_attention_heads": 8, "num_key_value_heads": 2, "head_dim": 128, "max_position_embeddings": 2048,
           "num_hidden_layers": 2}
    eng = Engine.from_random(config_from_dict(raw), seed=3, cache_dtype="float8_e4m3", max_tokens=4096, max_slots=4)
    rng = np.random.default_rng(3)
    p0, p1 = random_ids(rng, 1000, 256), random_ids(rng, 300, 256)

    def session(steps):
        s, t = eng.open(), eng.open()
        rows = [eng.step([StepEntry(s, p0, [0, 500, 999])]), eng.step([StepEntry(s, [7], [0]), StepEntry(t, p1, [299])])]
        for i in range(steps):
            rows.append(eng.step([StepEntry(s, [i], [0]), StepEntry(t, [2 * i], [0])]))
        assert eng.read_status() == 0
        eng.close(s)
        eng.close(t)
        return torch.cat(rows)

    first, replays = session(70), eng.graph_replays
    assert replays > 0 and torch.isfinite(first).all()
    assert torch.equal(session(70)[-2 * 60:], first[-2 * 60:])        # replayed in both sessions
    eng.use_graphs = False
    with monkeypatch.context() as m:
        calls = watch(eng, m)
        session(12)
        assert calls[0] == 14 * 2
