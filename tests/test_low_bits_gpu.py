"""Models that run with a cache of 8 bits and weights of 4, through the engine: against the plain formulas with the same codes."""
import pytest
import torch

import int8_cache_ref as ref
import plain_qwen2 as plain
from gpu_util import assert_close

pytestmark = pytest.mark.gpu


def engine(model_dir, page, dtype, num_pages=160, max_batch=4, **kw):
    from nanoinfer_b200.config import EngineConfig
    from nanoinfer_b200.engine import Engine
    return Engine(model_dir, EngineConfig(dtype=dtype, page_size=page, num_pages=num_pages, max_batch=max_batch, **kw))


def tokens(n, vocab, seed):
    return torch.randint(0, vocab, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def plain_rows(model, ids, portions, page):
    """Logits of one sequence that comes in portions, keys and values kept in 8 bits (page None: as they are), in 64 bits."""
    cfg, w = model.cfg, model.w
    pages = -(-len(ids) // (page or 1))
    cache = [[torch.zeros(pages, cfg["kv_heads"], page or 1, cfg["head_dim"], dtype=torch.float64) for _ in range(2)] for _ in range(cfg["layers"])]
    scales = [[torch.ones(pages, cfg["kv_heads"], dtype=torch.float64) for _ in range(2)] for _ in range(cfg["layers"])]
    out, at = [], 0
    for n in portions:
        pos = torch.arange(at, at + n)
        x = w["model.embed_tokens.weight"][torch.tensor(ids[at:at + n])]
        for i in range(cfg["layers"]):
            p = f"model.layers.{i}"
            window = cfg["window"] if (cfg["window"] and i >= cfg["max_window_layers"]) else 0
            h = plain.rms_norm(x, w[f"{p}.input_layernorm.weight"], cfg["eps"])
            q, k, v = (plain.linear(h, w[f"{p}.self_attn.{c}_proj.weight"], w.get(f"{p}.self_attn.{c}_proj.bias")).view(n, -1, cfg["head_dim"]) for c in "qkv")
            cos, sin = plain.rope_tables(pos, cfg["head_dim"], cfg["theta"])
            q, k = plain.apply_rope(q, cos, sin), plain.apply_rope(k, cos, sin)
            held = []
            for j, new in enumerate((k, v)):
                if page:
                    ref.append(cache[i][j], scales[i][j], new, at, list(range(pages)), page)
                    vals = ref.values(cache[i][j], scales[i][j])
                else:
                    cache[i][j][at:at + n, :, 0] = new
                    vals = cache[i][j]
                held.append(vals.permute(1, 0, 2, 3).reshape(cfg["kv_heads"], -1, cfg["head_dim"])[:, :at + n])
            rep = cfg["heads"] // cfg["kv_heads"]
            rows = torch.empty(n, cfg["heads"], cfg["head_dim"], dtype=torch.float64)
            for t in range(n):
                lo = max(0, at + t - window + 1) if window else 0
                for hd in range(cfg["heads"]):
                    kk, vv = held[0][hd // rep][lo:at + t + 1], held[1][hd // rep][lo:at + t + 1]
                    rows[t, hd] = torch.softmax(kk @ q[t, hd] * cfg["head_dim"] ** -0.5, dim=0) @ vv
            x = x + plain.linear(rows.reshape(n, -1), w[f"{p}.self_attn.o_proj.weight"])
            h = plain.rms_norm(x, w[f"{p}.post_attention_layernorm.weight"], cfg["eps"])
            x = x + plain.swiglu(h, w[f"{p}.mlp.gate_proj.weight"], w[f"{p}.mlp.up_proj.weight"], w[f"{p}.mlp.down_proj.weight"])
        x = plain.rms_norm(x, w["model.norm.weight"], cfg["eps"])
        out.append(plain.linear(x, w["model.embed_tokens.weight"] if cfg["tied"] else w["lm_head.weight"]))
        at += n
    return torch.cat(out)


def rms(x):
    return x.double().pow(2).mean().sqrt().item()


@pytest.mark.parametrize("name", ["A", "B", "W", "C"])
def test_8_bit_cache_in_32_bits_follows_the_plain_codes(model_dirs, name):
    """Portions and single tokens. In 32 bits a key that lies between two codes may take the other one: a few in a million, each worth
    a code; the rows must be far nearer to the plain model with the same codes than that one is to the model without them."""
    from nanoinfer_b200.engine import StepEntry
    d, page = model_dirs[name]
    model = plain.PlainModel(d)
    portions = [37, 1, 1, 20, 1, 1, 1, 9]
    ids = tokens(sum(portions), model.cfg["vocab"], 5)
    want, other = plain_rows(model, ids, portions, page), plain_rows(model, ids, portions, None)
    eng = engine(d, page, "float32", cache_dtype="int8")
    rc, at, got = eng.open("a"), 0, []
    for n in portions:
        got.append(eng.step([StepEntry(rc, ids[at:at + n], list(range(n)))]).clone())
        at += n
    got = torch.cat(got).cpu().double()
    assert rms(got - want) <= 0.1 * rms(want - other)
    eng.close(rc)
    eng.cache.check()


@pytest.mark.parametrize("name", ["B", "C"])
def test_8_bit_cache_in_bfloat16_decodes_replayed_and_eager_alike(model_dirs, name):
    """Two requests at different places, decoded by replayed graphs and without them: the same kernels on the same codes. Both stay
    within bfloat16's tolerance of the plain model with 8-bit codes (whose keys are not rounded to bfloat16 before)."""
    from nanoinfer_b200.engine import StepEntry
    d, page = model_dirs[name]
    model = plain.PlainModel(d)
    prompts, more = [tokens(61, model.cfg["vocab"], 6), tokens(18, model.cfg["vocab"], 7)], tokens(24, model.cfg["vocab"], 8)
    runs = []
    for graphs in (True, False):
        eng = engine(d, page, "bfloat16", cache_dtype="int8", cuda_graphs=graphs)
        rcs = [eng.open(i) for i in range(2)]
        rows = [eng.step([StepEntry(rc, p, [len(p) - 1]) for rc, p in zip(rcs, prompts)]).clone()]
        for t in range(0, 24, 2):
            rows.append(eng.step([StepEntry(rcs[0], [more[t]], [0]), StepEntry(rcs[1], [more[t + 1]], [0])]).clone())
        runs.append(torch.stack(rows))
        assert eng.graph_launches > 0 if graphs else eng.graph_launches == 0
        eng.check_device()
    assert torch.equal(runs[0], runs[1])
    for r in range(2):
        want = plain_rows(model, prompts[r] + more[r::2], [len(prompts[r])] + [1] * 12, page)
        assert_close(runs[0][:, r], want[len(prompts[r]) - 1:], torch.bfloat16, f"{name} request {r}")


def dequantized(model_dir, to, group):
    """The model folder with every matrix of attention and feed-forward replaced by what its 4-bit codes stand for."""
    import json
    import os
    import shutil
    from nanoinfer_b200.weights.int4 import Int4Matrix
    from nanoinfer_b200.weights.safetensors_io import save_safetensors
    from test_int4_cpu import unpacked
    w = plain.read_weights(model_dir, torch.float64)
    layers = sorted({k.split(".")[2] for k in w if k.startswith("model.layers.")}, key=int)
    for i in layers:
        for part, names in (("self_attn", ("q_proj", "k_proj", "v_proj")), ("self_attn", ("o_proj",)), ("mlp", ("gate_proj", "up_proj")), ("mlp", ("down_proj",))):
            keys = [f"model.layers.{i}.{part}.{n}.weight" for n in names]
            rows = unpacked(Int4Matrix.quantize(torch.cat([w[k] for k in keys]).float(), group))
            for k, r in zip(keys, rows.split([w[k].shape[0] for k in keys])):
                w[k] = r
    os.makedirs(to)
    shutil.copy(os.path.join(model_dir, "config.json"), to)
    save_safetensors(os.path.join(to, "model.safetensors"), {k: v.float().contiguous() for k, v in w.items()})


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name,group", [("A", 64), ("B", 64), ("C", 128)])
def test_4_bit_weights_are_the_model_with_their_values(model_dirs, tmp_path, name, group, dtype):
    from nanoinfer_b200.engine import StepEntry
    d, page = model_dirs[name]
    dequantized(d, str(tmp_path / "q"), group)
    model = plain.PlainModel(str(tmp_path / "q"))
    ids = tokens(140, model.cfg["vocab"], 9)
    want = model.logits(ids)
    eng = engine(d, page, dtype, weight_format="int4", weight_group=group)
    for portions in ([140], [70, 20, 1, 1, 40, 1, 7]):
        rc, at, got = eng.open("a"), 0, []
        for n in portions:
            got.append(eng.step([StepEntry(rc, ids[at:at + n], list(range(n)))]).clone())
            at += n
        assert_close(torch.cat(got), want[:at], torch.float32 if dtype == "float32" else torch.bfloat16, f"{name} {portions}")
        eng.close(rc)


def test_both_together_through_generation_and_the_scheduler(model_dirs):
    from nanoinfer_b200 import Request, Scheduler, load_model
    d, page = model_dirs["C"]
    model = load_model(d, page_size=page, num_pages=200, max_batch=4, max_tokens_per_step=64, cache_dtype="int8", weight_format="int4")
    prompts = [tokens(n, 1000, n) for n in (5, 90, 33, 170)]
    alone = [model.generate(p, max_tokens=12) for p in prompts]
    sched = Scheduler(model, lookahead=True)
    for i, p in enumerate(prompts):
        sched.add(Request(i, p, max_tokens=12))
    out = sched.run()
    assert all(len(alone[i]) == 12 and len(out[i]) == 12 for i in range(4))
    model.engine.cache.check()
    breakdown = model.weight_breakdown()
    assert breakdown["int4"][0] == 8 and model.engine.storage.bytes_per_token() == 2 * (2 * 2 * 64 + 1)


@pytest.mark.parametrize("weights", [None, 64])
def test_decoding_behind_prompts_of_hundreds_of_tokens(model_dirs, tmp_path, weights):
    """Contexts of several chunks of the decode kernel, whose earlier pages are sent for while the append still runs: logits of replayed and
    of eager steps against the plain model with the same codes, with weights of 16 bits and of 4. Replayed and eager are equal where both cut
    the keys alike: by themselves they choose 8 CTAs a row for the 1,024 keys that a graph is captured for and 4 for 534, whose sums of
    32 bits are of other terms. So the number is fixed; so is that of the prompt's products' parts of K, which add up as they come."""
    from nanoinfer_b200.config import KernelOptions
    from nanoinfer_b200.engine import StepEntry
    d, page = model_dirs["C"]
    kw = {}
    if weights:
        dequantized(d, str(tmp_path / "q"), weights)
        kw = dict(weight_format="int4", weight_group=weights)
    model = plain.PlainModel(str(tmp_path / "q") if weights else d)
    prompts = [tokens(n, model.cfg["vocab"], n) for n in (301, 140, 522)]
    more, steps = tokens(36, model.cfg["vocab"], 10), 12
    want = [plain_rows(model, p + more[r::3], [len(p)] + [1] * steps, page)[len(p) - 1:] for r, p in enumerate(prompts)]
    runs = []
    for graphs in (True, False):
        eng = engine(d, page, "bfloat16", num_pages=300, cache_dtype="int8", cuda_graphs=graphs, kernel_options=KernelOptions(fixed_decode_splits=4, tc_splits=1), **kw)
        rcs = [eng.open(i) for i in range(3)]
        rows = [eng.step([StepEntry(rc, p, [len(p) - 1]) for rc, p in zip(rcs, prompts)]).clone()]
        for t in range(steps):
            rows.append(eng.step([StepEntry(rc, [more[3 * t + r]], [0]) for r, rc in enumerate(rcs)]).clone())
        runs.append(torch.stack(rows))
        assert eng.graph_launches > 0 if graphs else eng.graph_launches == 0
        eng.check_device()
    assert torch.equal(runs[0], runs[1])
    for r in range(3):
        assert_close(runs[0][:, r], want[r], torch.bfloat16, f"request {r}")


def test_captured_portions_beside_decoded_tokens_follow_their_lengths(model_dirs):
    """A prompt fed in portions of 30 beside a request that decodes at 700 and on: replayed and eager steps give the same rows, and a graph's
    scratch is that of the power of two above the prompt's own context."""
    from nanoinfer_b200.config import KernelOptions
    from nanoinfer_b200.engine import StepEntry
    d, page = model_dirs["C"]
    model = plain.PlainModel(d)
    long, prompt, more = tokens(700, model.cfg["vocab"], 11), tokens(450, model.cfg["vocab"], 12), tokens(15, model.cfg["vocab"], 13)
    runs = []
    for graphs in (True, False):
        eng = engine(d, page, "bfloat16", num_pages=300, cache_dtype="int8", cuda_graphs=graphs, kernel_options=KernelOptions(fixed_decode_splits=4, tc_splits=1))
        if graphs:
            eng._portion_graphs.min_tokens, eng._portion_graphs.sightings = 16, 2
        a, b = eng.open("a"), eng.open("b")
        eng.step([StepEntry(a, long, [])])
        rows = []
        for t in range(15):
            rows.append(eng.step([StepEntry(b, prompt[30 * t:30 * t + 30], [29]), StepEntry(a, [more[t]], [0])]).clone())
        runs.append(torch.stack(rows))
        if graphs:
            captured = eng._portion_graphs.captured
            assert sorted(key[5] for key in captured) == [(256,), (512,)] and eng.graph_launches > 0
        eng.check_device()
    assert torch.equal(runs[0], runs[1])
    want = plain_rows(model, prompt, [30] * 15, page)[29::30]
    assert_close(runs[0][:, 0], want, torch.bfloat16, "the prompt")
    want = plain_rows(model, long + more, [700] + [1] * 15, page)[700:]
    assert_close(runs[0][:, 1], want, torch.bfloat16, "the decoded tokens")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_layer_that_reads_another_layers_8_bit_cache(tmp_path, dtype, monkeypatch):
    """A run order in which a layer reads the cache of an earlier one and writes none: its queries alone are rotated, and it sees the codes."""
    import test_toy_parts_gpu as toy
    from nanoinfer_b200.engine import StepEntry
    from nanoinfer_b200.registry import config_from_json_dict
    from nanoinfer_b200.weights import write_random_model
    toy._register()
    d, page = str(tmp_path / "toy"), 8
    write_random_model(config_from_json_dict(toy.TOY), d, seed=3)
    w, ids = toy.read_weights(d), tokens(61, 97, 14)
    other = toy.plain_toy(w, ids)

    def coded(x):
        pages = -(-x.shape[0] // page)
        codes, scales = torch.zeros(pages, x.shape[1], page, x.shape[2], dtype=torch.float64), torch.ones(pages, x.shape[1], dtype=torch.float64)
        ref.append(codes, scales, x, 0, list(range(pages)), page)
        return ref.values(codes, scales).permute(0, 2, 1, 3).reshape(-1, *x.shape[1:])[:x.shape[0]]

    attention = toy.causal_attention_fast
    monkeypatch.setattr(toy, "causal_attention_fast", lambda q, k, v: attention(q, coded(k), coded(v)))
    want = toy.plain_toy(w, ids)
    eng = engine(d, page, dtype, num_pages=40, max_batch=3, cache_dtype="int8")
    needs = eng.model.cache_needs()
    assert needs[4][0] is None and needs[4][2] == 1
    rc = eng.open("a")
    got = eng.step([StepEntry(rc, ids, list(range(61)))]).cpu().double()
    if dtype == "float32":
        assert rms(got - want) <= 0.1 * rms(want - other)
    else:
        assert_close(got, want, torch.bfloat16, "one portion")
    # decoded on: a token's own page is re-rounded as it fills, by less than a step, which is what the codes are from the plain model
    more = tokens(9, 97, 15)
    rows = torch.cat([eng.step([StepEntry(rc, [t], [0])]) for t in more]).cpu().double()
    want = toy.plain_toy(w, ids + more)[61:]
    monkeypatch.undo()
    assert rms(rows - want) <= 2 * rms(want - toy.plain_toy(w, ids + more)[61:]) + (0.015 * rms(want) if dtype == "bfloat16" else 0)
    eng.close(rc)
    eng.cache.check()
