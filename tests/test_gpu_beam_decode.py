"""Beam search over paged caches (beam_decode.py) against the context's own forward pass."""
import numpy as np
import pytest

import cpp_inference_train_engine_b200 as E
from cpp_inference_train_engine_b200.config import MLA36M, TINY
from tests.gpu_util import require_gpu

pytestmark = pytest.mark.gpu

# both sides' fp16 logits are held to these against the fp32 decoder (test_gpu_decode.py): twice that apart
TOL = {"tiny": 2 * 5e-3, "mla36m": 2 * 2e-2}
CONFIGS = {"tiny": TINY, "mla36m": MLA36M}
NEW = 9


def make(name, bits=16, beams=3, lens=(17, 1, 16), new=NEW, page=4, **kw):
    require_gpu()
    from cpp_inference_train_engine_b200.beam_decode import BeamDecoder
    cfg = CONFIGS[name]
    params = E.init_params(cfg, 3)
    rng = np.random.default_rng(4)
    prompts = [rng.integers(0, 256, n).tolist() for n in lens]
    return cfg, params, prompts, BeamDecoder(cfg, params, prompts, beams, new, page, bits, **kw)


def log_softmax(x):
    x = x.astype(np.float64)
    m = x.max(-1, keepdims=True)
    return x - m - np.log(np.exp(x - m).sum(-1, keepdims=True))


def score(ex, prompt, tokens):
    """Log-probability of `tokens` after `prompt` under the context's forward pass."""
    ids = np.array(prompt + tokens[:-1])
    lp = log_softmax(ex.forward(ids, 1, len(ids)))[len(prompt) - 1:]
    return float(sum(lp[i, t] for i, t in enumerate(tokens)))


def plain_search(ex, cfg, prompt, beams, new):
    """The same search, every hypothesis run through the forward pass anew."""
    alive = [([], 0.0)]
    for _ in range(new):
        cand = []
        for tokens, s in alive:
            if tokens and tokens[-1] == cfg.eos_id:
                cand.append((s, tokens))
                continue
            lp = log_softmax(ex.forward(np.array(prompt + tokens), 1, len(prompt) + len(tokens)))[-1]
            for t in np.argsort(-lp, kind="stable")[:beams]:
                cand.append((s + lp[t], tokens + [int(t)]))
        cand.sort(key=lambda c: -c[0])
        alive = [(t, s) for s, t in cand[:beams]]
    return alive


@pytest.mark.parametrize("name", CONFIGS)
@pytest.mark.parametrize("page", [4, 16])
def test_scores_are_the_forward_pass_log_probabilities(name, page):
    """Every hypothesis' score is its log-probability under the forward pass (a token's logits are TOL apart, and so
    is their log-sum-exp), and the best one is no worse than a plain search's by more than that."""
    cfg, params, prompts, d = make(name, page=page)
    ex = E.make_execution(cfg, params)
    out = d.search()
    for prompt, beams in zip(prompts, out):
        assert len(beams) == 3 and all(a[1] >= b[1] for a, b in zip(beams, beams[1:]))
        assert len({tuple(t) for t, _ in beams}) == 3
        for tokens, s in beams:
            assert 1 <= len(tokens) <= NEW and (len(tokens) == NEW or tokens[-1] == cfg.eos_id) and cfg.eos_id not in tokens[:-1]
            assert abs(s - score(ex, prompt, tokens)) <= 2 * TOL[name] * len(tokens)
        best = plain_search(ex, cfg, prompt, 3, NEW)[0]
        assert beams[0][1] >= best[1] - 4 * TOL[name] * NEW


@pytest.mark.parametrize("name", CONFIGS)
def test_one_beam_is_greedy(name):
    cfg, params, prompts, d = make(name, beams=1)
    ex = E.make_execution(cfg, params)
    for prompt, beams in zip(prompts, d.search()):
        tokens = beams[0][0]
        logits = ex.forward(np.array(prompt + tokens[:-1]), 1, len(prompt) + len(tokens) - 1)[len(prompt) - 1:]
        assert all(logits[i, t] >= logits[i].max() - 2 * TOL[name] for i, t in enumerate(tokens))


@pytest.mark.parametrize("name", CONFIGS)
def test_8_bit_pages_and_repeated_searches(name):
    """8-bit pages: scores follow from the decoder's own logits (a replay of the best hypothesis as a prompt's
    continuation). A second search gives the same bits."""
    cfg, params, prompts, d = make(name, bits=8)
    first, again = d.search(), d.search()
    assert first == again
    for g, beams in enumerate(first):
        tokens, s = beams[0]
        replay = make(name, bits=8, beams=1, lens=(17, 1, 16))[3]
        # one beam, its tokens given: the logits along the hypothesis
        import torch
        from cpp_inference_train_engine_b200 import paged
        prompts_of = torch.cat([replay.prompt_rows, replay.prompt_rows])  # every beam descends from its prompt's row
        table, spare, lengths = (t[:3] for t in paged.beam_reorder(replay.cache, *replay.start, prompts_of))
        total = float(torch.log_softmax(replay.prompt_logits[g].double(), -1)[tokens[0]])
        for i, t in enumerate(tokens[:-1]):
            step = torch.zeros(3, dtype=torch.int32, device="cuda")
            step[g] = t
            logits = replay.step_logits(step, lengths, table)
            lengths = lengths + 1
            total += float(torch.log_softmax(logits[g, 0].double(), -1)[tokens[i + 1]])
        # the rows of a product differ in the order of its sums by the number of rows alone
        assert abs(total - s) <= TOL[name] * len(tokens)


@pytest.mark.parametrize("page", [4, 16, 64])
@pytest.mark.parametrize("bits", [8, 16])
def test_searches_leave_the_prompts_as_they_were(page, bits):
    """A search's beams copy over each other's last pages: the next one finds the prompts' own untouched."""
    d = make("tiny", bits=bits, beams=5, page=page, new=20)[3]
    first = d.search()
    assert all(d.search() == first for _ in range(3))


def test_windowed_search():
    """A window that holds everything changes nothing but the order of the prompt's sums; a narrow one gives other
    scores and still ends."""
    cfg, _, prompts, d = make("mla36m")
    wide = make("mla36m", window=64)[3].search()
    for a, b in zip(d.search(), wide):
        assert abs(a[0][1] - b[0][1]) <= 4 * TOL["mla36m"] * NEW
    narrow = make("mla36m", window=3, sinks=1)[3].search()
    assert all(len(b) == 3 for b in narrow) and narrow[0][0][1] != wide[0][0][1]


def test_length_penalty_orders_the_beams():
    _, _, _, d = make("tiny")
    for beams in d.search(length_penalty=1.0):
        means = [s / len(t) for t, s in beams]
        assert all(a >= b - 1e-6 for a, b in zip(means, means[1:]))


def test_logits_without_a_token_are_an_error():
    cfg, params, prompts, d = make("tiny")
    d.embedding.fill_(float("nan"))
    d.prompt_logits.fill_(float("nan"))
    with pytest.raises(E.EngineError):
        d.search()


def test_command_reports_its_work(capsys):
    require_gpu()
    from cpp_inference_train_engine_b200 import beam_decode
    beam_decode.main(["--model", "tiny", "--requests", "2", "--beams", "3", "--prompt", "9", "--new", "5", "--cache-bits", "8"])
    assert "tokens/s" in capsys.readouterr().out
