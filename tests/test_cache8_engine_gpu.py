"""The 8-bit cache behind the framework's own paths: the attention mixer, the engine's steps and graphs, generation with a budget of rows,
the command line."""
import json
import math
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from conftest import ROOT, TINY
from plain import cache8_plain as plain
from test_parts_gpu import context_for, plain_weights, store_for

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H,G,D,window", [(4, 2, 64, 0), (6, 3, 32, 40), (5, 1, 48, 0), (16, 16, 128, 0), (7, 1, 128, 64)])
@pytest.mark.parametrize("q_lens,starts", [([70, 3], [0, 20]), ([1, 1], [100, 64])])
def test_the_mixer_writes_and_attends(dtype, H, G, D, window, q_lens, starts):
    """Its codes are those of its own projection (a product rounded to its type, so at most a step of the code beside the 64-bit one's), and its
    result is attention over what the codes stand for, then the output product."""
    from turboquant_cpp_b200.cache import PagedCache
    from turboquant_cpp_b200.csrc.build import ensure_built
    from turboquant_cpp_b200.parts import make_mixer, make_position_encoding
    hidden = 96
    mix = make_mixer("attention", prefix="a.", hidden=hidden, n_heads=H, n_kv_heads=G, head_dim=D, qkv_bias=True, window=window,
                     position=make_position_encoding("rotary", head_dim=D, theta=1e4, max_position=400, pairing="half"))
    mix.run_dtype, mix.cache8 = dtype, True
    store, specs = store_for(mix, 3, dtype)
    mix.bind(store)
    ensure_built(mix.kernels())
    assert {"cache8", "attention8", "evict"} <= set(mix.kernels())
    w = {k[2:].replace("_proj", ""): torch.from_numpy(v) for k, v in plain_weights(store, specs).items()}
    cache = PagedCache([mix.cache_need()], [None], [None], 1024, dtype, DEV, max_slots=4, eight_bits=True)
    runs = [n + s for n, s in zip(q_lens, starts)]
    x = torch.randn(sum(runs), hidden).to(dtype)
    seqs, at = [], 0
    pieces = []
    for n, s in zip(q_lens, starts):                    # the rows held already, written by steps of their own
        pieces.append(x[at:at + s + n])
        at += s + n
    tables = None
    ctx, tables, seqs = context_for(q_lens, [0, 0], dtype, cache)
    for seq in seqs:
        cache.close(seq)
    seqs = [cache.open() for _ in q_lens]
    for step, lens in ((0, starts), (1, q_lens)):
        todo = [i for i, n in enumerate(lens) if n]
        if not todo:
            continue
        ns = [lens[i] for i in todo]
        cache.reserve([seqs[i] for i in todo], ns)
        first = [seqs[i].length for i in todo]
        cu = np.concatenate([[0], np.cumsum(ns)])
        i32 = lambda a: torch.tensor(np.asarray(a), dtype=torch.int32, device=DEV)
        ctx.n_tokens, ctx.n_seqs, ctx.cu_seqlens, ctx.seq_start, ctx.max_q_len = sum(ns), len(ns), i32(cu), i32(first), max(ns)
        ctx.seq_of_token = i32(np.repeat(np.arange(len(ns)), ns))
        ctx.positions = i32(np.concatenate([np.arange(n) + f for n, f in zip(ns, first)]))
        ctx.max_kv_len = max(a + b for a, b in zip(first, ns))
        xs = torch.cat([pieces[i][seqs[i].length:seqs[i].length + lens[i]] for i in todo]).to(DEV)
        table = i32(cache.page_tables([seqs[i] for i in todo])[0])
        got = mix.forward(xs, ctx, cache.layer_caches([table])[0]).double().cpu()
        cache.commit([seqs[i] for i in todo], ns)
    codes, scales = cache.kv[0].view(torch.uint8).cpu(), cache.scales[0].cpu()
    table = torch.from_numpy(cache.page_tables(seqs)[0])
    i = torch.arange(D // 2, dtype=torch.float64)
    want, mags, limits = [], [], []
    for s, (n, start) in enumerate(zip(q_lens, starts)):
        xs = pieces[s].double()
        angle = torch.arange(n + start)[:, None] * torch.pow(1e4, -2 * i / D)
        heads = lambda name, k: (xs @ w[name + ".weight"].T + w[name + ".bias"]).view(n + start, k, D)
        turn = lambda t: plain.rotate(t, torch.cos(angle), torch.sin(angle), "half")
        q, k, v = turn(heads("q", H)), turn(heads("k", G)), heads("v", G)
        first = max(0, n + start + 1 - (window or 10 ** 6)) // 64 * 64            # pages behind the window were given back
        got_k, got_v = plain.rows_of(codes, scales, table, s, n + start, 64)
        unit = torch.finfo(dtype).eps
        for mine, theirs in ((got_k, k), (got_v, v)):
            theirs = theirs.transpose(0, 1)[:, first:]
            top = theirs.abs().amax((1, 2), keepdim=True)
            # the projection rounded to its type, then at most half a step of the code (a block's smallest step: 2^-17 of its largest)
            assert bool(((mine[:, first:] - theirs).abs() <= 2.0 ** -4 * theirs.abs() * 1.001 + (2.0 ** -17 + 4 * unit) * top).all())
        out, mag, units, _ = plain.attention(q[start:].to(dtype).double().reshape(n, H, D), codes, scales, [n], [start], table[s:s + 1], 64, window, 1 / math.sqrt(D), H, G, D)
        # queries rounded to their type move a score by up to eps of its products' magnitudes (projection and rotation: two roundings each way)
        rel = (2 * unit + (D + 8) * 2.0 ** -22) * 2.02 * units[..., None] + (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -20)
        limits.append((rel * mag + unit * out.abs()).reshape(n, -1) @ w["o.weight"].abs().T)
        mags.append(mag.reshape(n, -1) @ w["o.weight"].abs().T)
        want.append(out.reshape(n, -1) @ w["o.weight"].T)
    want, limit = torch.cat(want), torch.cat(limits) + torch.cat(mags) * 2.0 ** -18
    assert bool(((got - want).abs() <= limit).all()), float(((got - want).abs() / limit).max())


@pytest.fixture(scope="module")
def model_of(tiny_folders):
    import turboquant_cpp_b200 as tq
    made = {}

    def get(name, dtype="float32"):
        if (name, dtype) not in made:
            made[name, dtype] = tq.load_model(tiny_folders[name], dtype, DEV)
        return made[name, dtype]
    return get


def _logits(engine, tokens, cuts):
    """Logits of every token, the request cut into steps of these lengths."""
    import turboquant_cpp_b200 as tq
    seq, out, at = engine.open(), [], 0
    for n in cuts:
        out.append(engine.step([tq.StepEntry(seq, tokens[at:at + n], list(range(n)))]).cpu())
        at += n
    engine.close(seq)
    return torch.cat(out)


@pytest.mark.parametrize("name", ["A", "B", "C"])
def test_logits_do_not_depend_on_the_cut(model_of, name):
    """A block's byte grows as rows come: what was written under a smaller one is rounded again, which moves codes below e4m3's normal range
    only, by at most 2^-17 of the block's largest magnitude.  Everything else is float32; through the layers that is far below 2e-3 of
    the logits' scale unless a router's choice flips (which these seeds do not meet)."""
    import turboquant_cpp_b200 as tq
    engine = tq.Engine(model_of(name), max_tokens=512, cache_dtype="e4m3")
    V = TINY[name][0]["vocab_size"]
    tokens = np.random.default_rng(5).integers(0, V, size=110).tolist()
    whole = _logits(engine, tokens, [110])
    for cuts in ([50, 60], [1] * 20 + [90], [70] + [1] * 40):
        got = _logits(engine, tokens, cuts)
        off = (got - whole).abs().amax(1) / whole.abs().max()
        assert float(off.max()) < 2e-3, (cuts, float(off.max()))
    engine.cache.book.check_invariants()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_graphs_replay_what_plain_steps_compute(model_of, dtype):
    import turboquant_cpp_b200 as tq
    out = []
    for graphs in (False, True):
        engine = tq.Engine(model_of("A", dtype), max_tokens=1024, cache_dtype="e4m3", cache_budget=32, cache_recent=8, use_graphs=graphs)
        seqs = [engine.open() for _ in range(3)]
        engine.step([tq.StepEntry(s, list(range(5 + 30 * i))) for i, s in enumerate(seqs)])
        rows = [engine.step([tq.StepEntry(s, [7 * t % 256], [0]) for s in seqs]).cpu() for t in range(50)]
        assert all(s.held < 96 for s in seqs) and seqs[2].evicted > 0 and seqs[2].length == 115
        engine.cache.book.check_invariants()
        out.append((torch.stack(rows), [w.cpu() for w in engine.cache.weights], [s.held for s in seqs]))
        for s in seqs:
            engine.close(s)
        engine.cache.book.check_invariants()
        engine.release()
    assert torch.equal(out[0][0], out[1][0]) and out[0][2] == out[1][2]
    assert all(torch.equal(a, b) for a, b in zip(out[0][1], out[1][1]))


def test_an_evicted_sequence_goes_on_from_the_rows_it_keeps(model_of):
    """Two engines step the same tokens; one evicts, keeping the newest rows only.  A third starts from a cache whose tables the test sets to those
    rows by hand: the first one's logits are the third's."""
    import turboquant_cpp_b200 as tq
    model = model_of("A")
    tokens = np.random.default_rng(8).integers(0, 256, size=100).tolist()
    evicting = tq.Engine(model, max_tokens=512, cache_dtype="e4m3", cache_budget=32, cache_recent=32, use_graphs=False)
    a = evicting.open()
    evicting.step([tq.StepEntry(a, tokens[:96])])
    assert (a.held, a.evicted, a.length) == (32, 64, 96)
    got = evicting.step([tq.StepEntry(a, [tokens[96]], [0])]).cpu()
    # places 64 .. 95 of a sequence that kept all are the first 32 of a page: a sequence that has this page alone holds just those rows
    keeping = tq.Engine(model, max_tokens=512, cache_dtype="e4m3", use_graphs=False)
    b = keeping.open()
    keeping.step([tq.StepEntry(b, tokens[:96])])
    for g in range(len(b.pages)):
        for p in b.pages[g][:-1]:
            keeping.cache.book.pools[g].give_back(p)
        b.pages[g] = b.pages[g][-1:]
    b.evicted = 64
    want = keeping.step([tq.StepEntry(b, [tokens[96]], [0])]).cpu()
    assert torch.equal(got, want)


def test_generation_with_a_budget(model_of):
    import turboquant_cpp_b200 as tq
    model = model_of("A")
    prompts = [[5, 9, 2], list(range(60)), [1] * 20, [200, 100]]
    run = lambda **kw: _generate(tq, model, prompts, **kw)
    plain8, stats = run(cache_dtype="e4m3")
    never, _ = run(cache_dtype="e4m3", cache_budget=128)               # a request has at most 128 tokens: nothing is evicted
    assert never == plain8
    bounded, stats = run(cache_dtype="e4m3", cache_budget=24, cache_recent=6)
    assert [len(t) for t in bounded] == [len(t) for t in plain8] and bounded != plain8
    assert bounded == run(cache_dtype="e4m3", cache_budget=24, cache_recent=6)[0]
    assert bounded[1:2] == _generate(tq, model, prompts[1:2], cache_dtype="e4m3", cache_budget=24, cache_recent=6)[0]


def _generate(tq, model, prompts, **kw):
    with tq.Model.from_model(model, temperature=0.0, max_tokens=60, context_length=128, max_batch=4, stop_token_ids=[], **kw) as m:
        out = m.generate_batch(prompts)
        m.engine.cache.book.check_invariants()
        per = m.engine.cache.bytes_per_token()
        # two layers of 4 key/value heads of 16: codes of two planes, 2 x 4 bytes for 16 rows, a float a head and row
        assert per == 2 * (2 * 4 * 16) + 2 * (2 * 4) // 16 + (2 * 4 * 4 if kw.get("cache_budget") else 0)
        return out, m.last_stats


def test_the_command_line(tmp_path, tiny_folders):
    run = lambda *more: subprocess.run([sys.executable, os.path.join(ROOT, "bin", "quant"), tiny_folders["A"], "-p", "1,2,3", "-n", "100", "-T", "0", "--stop", "-1",
                                        "--dtype", "float32", *more], capture_output=True, text=True, timeout=300)
    full, bounded = run("--cache", "e4m3"), run("--cache", "e4m3", "--cache-budget", "16", "--cache-recent", "4")
    for r in (full, bounded):
        assert r.returncode == 0, r.stderr
    assert len(full.stdout.split()) == len(bounded.stdout.split()) == 100 and full.stdout != bounded.stdout
    refused = run("--cache-budget", "16")
    assert refused.returncode != 0 and "cache_budget needs a cache in 8 bits" in refused.stderr
