"""Forked sequences, several answers to a prompt, log probabilities and scores through the engine: every architecture's forks
against the same sequences run on their own, generation against the plain implementation."""
import importlib
import math
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import helpers
from plain_lfm2 import PlainLfm2

pytestmark = pytest.mark.gpu

ARCHS = ["kerotar", "pirisun", "ponusun", "varolorn", "zosurax", "nipizen"]


@pytest.fixture(scope="module")
def zoo(tmp_path_factory):
    """(architecture, name) -> folder, of every test configuration of the later architectures."""
    root = tmp_path_factory.mktemp("fork_models")
    out = {}
    for arch in ARCHS:
        H = importlib.import_module(arch + "_helpers")
        for i, (name, cfg) in enumerate(H.CONFIGS.items()):
            W = (H.make_weights(name, 40 + i) if arch == "varolorn" else H.make_weights(cfg, 40 + i, H.RANKS[name]) if arch == "nipizen"
                 else H.make_weights(cfg, 40 + i))
            out[arch, name] = H.write_folder(root / arch / name, cfg, W)
    return out


def shared_always(engine):
    engine.MIN_KEYS_SAVED, engine.MIN_SHARE_SAVED = 1, 0.0
    for part in engine.model.all_parts():
        if hasattr(part, "general_min_saved"):
            part.general_min_saved = 0
    return engine


def forks_and_alone(engine, prompt, n, steps, seed, decode=True):
    """Logits of `steps` single-token steps of n forks of a prompt, and of the same sequences run on their own."""
    vocab = engine.vocab_size
    feed = np.random.default_rng(seed).integers(0, vocab, size=(steps, n)).tolist()
    got, want = [], []
    for forked in (True, False):
        if forked:
            s, = engine.start(1)
            engine.step([s], [prompt])
            slots = [s, *engine.fork(s, n - 1)]
        else:
            slots = engine.start(n)
            engine.step(slots, [prompt] * n)
        for row in feed:
            x = engine.decode(slots, row, check=True) if decode else engine.step(slots, [[t] for t in row])
            (got if forked else want).append(x.cpu().numpy().copy())
        engine.cache.check_consistency()
        if forked:
            assert bool(engine.cache.shared_prefixes(slots)) == any(
                g.request.window <= 0 and g.request.chunk <= 0 and len(prompt) >= g.page_size for g in engine.cache.groups)
        engine.finish(slots)
    assert engine.cache.free_page_count() == [g.num_pages for g in engine.cache.groups]
    return np.stack(got), np.stack(want)


def all_models():
    out = []
    for arch in ARCHS:
        H = importlib.import_module(arch + "_helpers")
        out += [(arch, name) for name in H.CONFIGS]
    return out


@pytest.mark.parametrize("arch,name", all_models())
def test_forks_of_every_architecture(zoo, arch, name):
    """In 32 bits the forks' logits are those of sequences of their own, up to the order of sums (twice the bound that either keeps
    against the plain implementation)."""
    import zinfer_b200 as z
    model = z.load(zoo[arch, name], dtype="fp32")
    longest = min(model.config.max_position_embeddings, 256)
    engine = shared_always(z.Engine(model, max_batch=4, max_seq_len=longest, page_size=16))
    prompt = helpers.random_tokens(3, min(100, longest - 12), engine.vocab_size)
    got, want = forks_and_alone(engine, prompt, 4, 8, 5)
    assert helpers.rel_err(got, want) <= 2 * 5e-5


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", helpers.LOUD)
def test_forks_of_lfm2(model_folders, name, dtype):
    import zinfer_b200 as z
    engine = shared_always(z.Engine(z.load(model_folders[name], dtype=dtype), max_batch=6, max_seq_len=128,
                                    page_size=64 if name in ("loud_d", "loud_e") else 16))
    for length, n in ((100, 6), (64, 2), (15, 3), (1, 2)):
        for decode in (True, False):
            got, want = forks_and_alone(engine, helpers.random_tokens(length, length, engine.vocab_size), n, 5, length, decode)
            assert helpers.rel_err(got, want) <= 2 * helpers.tol(name, dtype)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("head_dim", [256, 258, 320])
def test_forks_of_heads_wider_than_the_shared_kernels_take(dtype, head_dim):
    """Heads of more than 256 decode from forks as they do alone: each reads what it shares for itself."""
    import zinfer_b200 as z
    cfg = dict(helpers.TINY["loud_a"]["config"], head_dim=head_dim)
    engine = shared_always(z.Engine(z.random(cfg, seed=3, dtype=dtype, std=0.125), max_batch=4, max_seq_len=128, page_size=16))
    assert engine._takes_prefixes == (head_dim <= 256)
    prompt = helpers.random_tokens(7, 70, engine.vocab_size)
    for decode in (True, False):
        got, want = forks_and_alone(engine, prompt, 4, 5, 9, decode)
        assert helpers.rel_err(got, want) <= 2 * helpers.tol("loud_a", dtype)
    answers, = engine.generate([prompt], max_new_tokens=6, temp=0.0, stop_ids=[], samples=3)
    alone, = engine.generate([prompt], max_new_tokens=6, temp=0.0, stop_ids=[])
    assert [len(a.tokens) for a in answers] == [6] * 3 and (dtype == "bfloat16" or all(a.tokens == alone.tokens for a in answers))


def test_long_shared_prefix_on_the_tensor_cores(model_folders):
    """More pairs than 32 to a KV head and a prefix over several blocks: the tcgen05 kernel beside the single sequences' one, recorded
    and replayed over the steps at which layouts change, with sequences that end and others among them."""
    import zinfer_b200 as z
    name = "loud_d"
    engine = shared_always(z.Engine(z.load(model_folders[name], dtype="bf16"), max_batch=24, max_seq_len=900, page_size=64))
    vocab = engine.vocab_size
    rng = np.random.default_rng(1)
    prompt, other = rng.integers(0, vocab, 700).tolist(), rng.integers(0, vocab, 90).tolist()
    feed = rng.integers(0, vocab, size=(140, 24)).tolist()
    runs = []
    for forked in (True, False):
        if forked:
            a, b = engine.start(2)
            engine.step([a, b], [prompt, other])
            slots = [a, *engine.fork(a, 19)] + [b, *engine.fork(b, 3)]
        else:
            slots = engine.start(24)
            engine.step(slots, [prompt] * 20 + [other] * 4)
        out = []
        for i, row in enumerate(feed):
            live = list(range(24)) if i < 100 else list(range(3, 24, 2))
            x = engine.decode([slots[j] for j in live], [row[j] for j in live], check=i % 20 == 0)
            if i % 9 == 0 or i in (98, 99, 100, 101, 139):
                out.append(x.cpu().numpy().copy())
        engine.check_status()
        engine.cache.check_consistency()
        engine.finish(slots)
        runs.append(out)
    assert any("shared" in key for key in engine._graphs)
    for got, want in zip(*runs):
        assert helpers.rel_err(got, want) <= 2 * helpers.tol(name, "bfloat16")


@pytest.mark.parametrize("name,dtype,page", [("loud_d", "bf16", 64), ("loud_c", "fp32", 16)])
def test_steps_of_forks_are_prepared(model_folders, name, dtype, page):
    """Recorded ahead for sequences that share prefixes, over the lengths at which their launches change, until sharing no longer pays;
    a batch that has run shared steps alone has none without prefixes to record, and says so."""
    import zinfer_b200 as z
    prompt = helpers.random_tokens(1, 3 * page + 9, 256)
    feed = np.random.default_rng(2).integers(0, 256, size=(290, 6)).tolist()
    runs = []
    for prepared in (True, False):
        engine = shared_always(z.Engine(z.load(model_folders[name], dtype=dtype), max_batch=6, max_seq_len=512, page_size=page))
        engine.MIN_SHARE_SAVED = 0.41 if page == 64 else 0.15        # some 200 tokens on the answers' own keys outweigh the prompt
        s, = engine.start(1)
        engine.step([s], [prompt])
        slots = [s, *engine.fork(s, 5)]
        first = engine.length(s) + 1
        if prepared:
            with pytest.raises(RuntimeError, match="with these shared prefixes"):
                engine.prepare_decode(6, first, first + 150, slots=slots)
        engine.decode(slots, feed[0])
        if prepared:
            with pytest.raises(RuntimeError, match="without shared prefixes"):
                engine.prepare_decode(6, first, first + 150)
            with pytest.raises(ValueError):
                engine.prepare_decode(5, first, first + 150, slots=slots)
            engine.prepare_decode(6, first + 1, first + 150, slots=slots)
            before = engine.graph_captures
            assert before >= 2                                        # own keys up to 128, and up to 192
        out = []
        for i in range(1, 290):
            x = engine.decode(slots, feed[i], check=i % 50 == 0)
            if prepared and i == 150:
                assert engine.graph_captures == before                # every step of the range was there
            if i % 17 == 0:
                out.append(x.cpu().numpy().copy())
        assert not engine.shared_prefixes(slots) and engine._decode_batches[6].warmed
        if prepared:
            engine.prepare_decode(6, first + 290, first + 292, slots=slots)      # by now they share nothing that pays
        engine.check_status()
        runs.append(out)
    for got, want in zip(*runs):
        assert np.array_equal(got, want)


def test_sharing_is_used_where_it_pays(model_folders):
    import zinfer_b200 as z
    engine = z.Engine(z.load(model_folders["tiny_d"], dtype="bf16"), max_batch=10, max_seq_len=1000, page_size=64)
    prompt = helpers.random_tokens(1, 650, engine.vocab_size)
    s, = engine.start(1)
    engine.step([s], [prompt])
    forks = engine.fork(s, 9)
    assert engine.shared_prefixes([s, *forks]) == [(list(range(10)), 640)]
    assert engine.shared_prefixes([s, *forks[:5]]) == []             # 5 x 640 keys
    assert engine.shared_prefixes(forks[:8]) == [(list(range(8)), 640)]
    engine.finish(forks[:7])
    assert engine.shared_prefixes([s, *forks[7:]]) == []


def test_a_fork_does_not_change_the_sequence_it_came_from(model_folders):
    import zinfer_b200 as z
    engine = shared_always(z.Engine(z.load(model_folders["loud_c"], dtype="fp32"), max_batch=3, max_seq_len=256, page_size=16))
    vocab = engine.vocab_size
    prompt, tail = helpers.random_tokens(1, 90, vocab), helpers.random_tokens(2, 30, vocab)
    s, = engine.start(1)
    engine.step([s], [prompt])
    f, = engine.fork(s, 1)
    engine.step([f], [helpers.random_tokens(3, 100, vocab)])         # a long step of the fork alone
    got = engine.step([s], [tail], want=[list(range(30))]).cpu().numpy()
    engine.finish([f])
    g, = engine.fork(s, 1)                                           # pages of the first fork are used again
    more = engine.step([g, s], [[5], [5]]).cpu().numpy()
    engine.finish([s, g])
    alone, = engine.start(1)
    want = engine.step([alone], [prompt + tail + [5]], want=[list(range(90, 121))]).cpu().numpy()
    assert helpers.rel_err(got, want[:30]) <= 1e-4
    assert helpers.rel_err(more, want[[30, 30]]) <= 1e-4


def test_errors_of_a_fork_leave_the_engine_as_it_was(model_folders):
    import zinfer_b200 as z
    from zinfer_b200.cache import NoFreeSlot, OutOfPages
    engine = z.Engine(z.load(model_folders["tiny_a"], dtype="fp32"), max_batch=3, max_seq_len=64, max_tokens=64, page_size=16)
    s, = engine.start(1)
    engine.step([s], [helpers.random_tokens(1, 50, engine.vocab_size)])
    with pytest.raises(OutOfPages):
        engine.fork(s, 1)
    with pytest.raises(NoFreeSlot):
        engine.fork(s, 3)
    engine.cache.check_consistency()
    engine.decode([s], [3], check=True)


@pytest.mark.parametrize("name", ["loud_a", "loud_d"])
def test_several_greedy_answers_are_the_plain_one(model_folders, name):
    import zinfer_b200 as z
    plain = PlainLfm2(model_folders[name], dtype=np.float64)
    engine = shared_always(z.Engine(z.load(model_folders[name], dtype="fp32"), max_batch=5, max_seq_len=128, page_size=16))
    prompts = [helpers.random_tokens(10 + i, n, engine.vocab_size) for i, n in enumerate([40, 3, 17])]
    results = engine.generate(prompts, max_new_tokens=10, temp=0.0, stop_ids=[], samples=3)
    assert [len(r) for r in results] == [3, 3, 3]
    for p, answers in zip(prompts, results):
        assert all(r.tokens == plain.greedy(p, 10)[0] for r in answers)
    assert engine.cache.free_slot_count() == 5
    engine.cache.check_consistency()


def test_sampled_answers_are_those_of_single_requests(model_folders):
    """Answer j to prompt i is request i * n + j: its random numbers do not depend on whether the prompt was run for it."""
    import zinfer_b200 as z
    engine = shared_always(z.Engine(z.load(model_folders["tiny_b"], dtype="fp32"), max_batch=8, max_seq_len=128, page_size=16))
    prompts = [helpers.random_tokens(20 + i, n, engine.vocab_size) for i, n in enumerate([30, 5])]
    for options in (dict(temp=1.0, seed=3), dict(temp=0.9, seed=4, repeat_penalty=1.3), dict(temp=0.9, seed=5, dry_multiplier=0.8)):
        many = engine.generate(prompts, max_new_tokens=12, stop_ids=[], samples=4, **options)
        alone = engine.generate([p for p in prompts for _ in range(4)], max_new_tokens=12, stop_ids=[], **options)
        assert [r.tokens for a in many for r in a] == [r.tokens for r in alone]
        assert len({tuple(r.tokens) for r in many[0]}) > 1


def check_scores(scores, tokens, logits, tol, top):
    """`logits`: the plain implementation's at the positions before the tokens.  A log probability moves by at most twice what the
    logits do, an entropy by that times the spread of the log probabilities under the distribution."""
    m = logits.max(axis=1, keepdims=True)
    lp = logits - m - np.log(np.exp(logits - m).sum(axis=1, keepdims=True))
    off = tol * np.abs(logits).max()
    p = np.exp(lp)
    assert len(scores.logprobs) == len(scores.ranks) == len(scores.entropies) == len(tokens)
    for i, t in enumerate(tokens):
        assert abs(scores.logprobs[i] - lp[i, t]) <= 2 * off + 1e-5
        sure = int((lp[i] > lp[i, t] + 4 * off).sum())
        assert 1 + sure <= scores.ranks[i] <= int((lp[i] >= lp[i, t] - 4 * off).sum())
        h = -(p[i] * lp[i]).sum()
        spread = math.sqrt(max(0.0, (p[i] * lp[i] ** 2).sum() - h * h))
        assert abs(scores.entropies[i] - h) <= 2 * off * (spread + 2 * off) * math.exp(4 * off) + 1e-5
        if top:
            assert len(scores.top[i]) == top and len({k for k, _ in scores.top[i]}) == top
            best = np.sort(lp[i])[::-1]
            for j, (k, v) in enumerate(scores.top[i]):
                assert abs(v - lp[i, k]) <= 2 * off + 1e-5 and abs(v - best[j]) <= 2 * off + 1e-5


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_generated_log_probabilities(model_folders, dtype):
    """Greedy, sampled and penalised tokens, steps that run ahead and steps that do not; stop tokens; one answer and several."""
    import zinfer_b200 as z
    name = "loud_a"
    plain = PlainLfm2(model_folders[name], dtype=np.float64)
    prompts = [helpers.random_tokens(30 + i, n, 256) for i, n in enumerate([25, 4, 60])]
    for lookahead in (True, False):
        engine = shared_always(z.Engine(z.load(model_folders[name], dtype=dtype), max_batch=4, max_seq_len=128, page_size=16,
                                        lookahead=lookahead, use_graphs=lookahead))
        probe = engine.generate(prompts, max_new_tokens=8, temp=0.0, stop_ids=[])
        stop = [probe[1].tokens[5]]
        for options in (dict(temp=0.0, samples=2), dict(temp=0.7, seed=1), dict(temp=0.0, repeat_penalty=1.5), dict(temp=1.0, seed=2, dry_multiplier=1.0)):
            for top in (0, 3):
                results = engine.generate(prompts, max_new_tokens=8, stop_ids=stop, logprobs=top, **options)
                if "samples" in options:
                    results, owners = [r for a in results for r in a], [p for p in prompts for _ in range(2)]
                else:
                    owners = prompts
                for p, r in zip(owners, results):
                    seen = r.tokens + ([r.stop_token] if r.stop_token is not None else [])
                    ref = plain.logits(p + seen)[len(p) - 1:len(p) - 1 + len(seen)]
                    check_scores(r.logprobs, seen, ref, helpers.tol(name, dtype), top)
                    if options == dict(temp=0.0, samples=2):
                        assert r.logprobs.ranks == [1] * len(seen)
        with pytest.raises(ValueError):
            engine.generate(prompts, logprobs=33)
        with pytest.raises(ValueError):
            engine.generate(prompts, samples=0)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["loud_a", "loud_c"])
def test_scores_of_given_tokens(model_folders, name, dtype):
    import zinfer_b200 as z
    plain = PlainLfm2(model_folders[name], dtype=np.float64)
    vocab = plain.cfg["vocab_size"]
    engine = z.Engine(z.load(model_folders[name], dtype=dtype), max_batch=3, max_seq_len=128, page_size=16, max_step_tokens=50)
    seqs = [helpers.random_tokens(70 + i, n, vocab) for i, n in enumerate([2, 128, 1, 33, 90, 7])]
    for top in (0, 5):
        scores = engine.score(seqs, top)
        for s, r in zip(seqs, scores):
            if len(s) == 1:
                assert r == z.TokenScores()
            else:
                check_scores(r, s[1:], plain.logits(s)[:-1], helpers.tol(name, dtype), top)
    assert engine.cache.free_slot_count() == 3
    for bad in ([[]], [[1, vocab]], [[-1, 2]], [list(range(1)) * 130]):
        with pytest.raises(ValueError):
            engine.score(bad)
    with pytest.raises(ValueError):
        engine.score(seqs, 33)


def test_the_command_line(model_folders):
    folder = model_folders["loud_a"]
    plain = PlainLfm2(folder, dtype=np.float64)
    prompt = helpers.random_tokens(90, 20, 256)

    def run(*args):
        proc = subprocess.run([str(helpers.ROOT / "bin" / "zinfer_b200"), "-m", str(folder), "-p", ",".join(map(str, prompt)), "--dtype", "fp32",
                               "--stop", "", *map(str, args)], capture_output=True, text=True, timeout=600,
                              env=dict(os.environ, ZINFER_PYTHON=sys.executable))
        assert proc.returncode == 0, proc.stderr[-3000:]
        return proc.stdout.strip().splitlines()

    want = plain.greedy(prompt, 5)[0]
    lines = run("-n", 5, "--temp", 0, "--samples", 3)
    assert lines == [" ".join(map(str, want)) + "  [length]"] * 3
    ref = plain.logits(prompt + want)
    lp = ref - ref.max(axis=1, keepdims=True)
    lp = lp - np.log(np.exp(lp).sum(axis=1, keepdims=True))
    line, = run("-n", 5, "--temp", 0, "--logprobs", 2)
    for i, part in enumerate(line.replace("  [length]", "").replace(") ", ")\n").split("\n")):
        head, top = part.rstrip(")").split("(")
        token, rest = head.split(":")
        value, rank = rest.split("#")
        assert int(token) == want[i] and rank == "1" and abs(float(value) - lp[len(prompt) - 1 + i, want[i]]) < 1e-3
        assert len(top.split()) == 2 and top.split()[0].startswith(token + ":")
    line, = run("--score")
    total, tokens = line.split("  ", 1)
    parts = [lp[i, t] for i, t in enumerate(prompt[1:])]
    assert abs(float(total) - sum(parts)) < 0.01 and [int(t.split(":")[0]) for t in tokens.split()] == prompt[1:]
