"""Beam search where kernels fail, hypotheses end early, and the prompt is seen through a window."""
import numpy as np
import pytest

import cpp_inference_train_engine_b200 as E
from tests.gpu_util import require_gpu
from tests.test_gpu_beam_decode import make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("module", ["latent", "paged"])
def test_a_kernel_that_gave_up_is_reported_as_such(module, monkeypatch):
    """The status that the device keeps is asked for after the prompts, at a search's end, and before a missing
    continuation is blamed on the logits: here a fake one that says yes."""
    require_gpu()
    from cpp_inference_train_engine_b200 import latent, paged
    asked = []

    def gave_up(device=None):
        asked.append(device)
        raise E.EngineError(5, "a kernel gave up")

    d = make("tiny")[3]
    with monkeypatch.context() as m:
        m.setattr({"latent": latent, "paged": paged}[module], "check_status", gave_up)
        with pytest.raises(E.EngineError, match="gave up"):
            make("tiny")
        with pytest.raises(E.EngineError, match="gave up"):
            d.search()
        kept = d.prompt_logits.clone()
        d.prompt_logits.fill_(float("nan"))
        with pytest.raises(E.EngineError, match="gave up"):
            d.search()
        d.prompt_logits.copy_(kept)
    assert asked == [d.device] * 3
    assert len(d.search()) == 3


# ------------------------------------------------------------------ hypotheses that end
def ending(cfg, params, share=0.6):
    """Parameters under which hypotheses end at different steps: logits four times as large (final norm), and an end-of-sequence
    row that lies along every seventh token's, so that it is likely after those."""
    params = params.copy()
    V, d = cfg.vocab_size, cfg.d_model
    emb = params[:V * d].reshape(V, d)
    emb[cfg.eos_id] = share * emb[:256:7].sum(0)
    params[V * d:V * d + d] *= 4
    return params


def make_ending(bits, page, beams=4, lens=(17, 1, 16), new=9, share=0.6):
    require_gpu()
    from cpp_inference_train_engine_b200.beam_decode import BeamDecoder
    from cpp_inference_train_engine_b200.config import TINY
    params = ending(TINY, E.init_params(TINY, 3), share)
    rng = np.random.default_rng(4)
    prompts = [rng.integers(0, 256, n).tolist() for n in (17, 1, 16)]
    prompts = [p for p in prompts if len(p) in lens]
    return TINY, params, prompts, BeamDecoder(TINY, params, prompts, beams, new, page, bits)


def recorded(d):
    """The logits of a search's steps, as the decoder makes them."""
    steps, step = [], d.step_logits
    d.step_logits = lambda *a: steps.append(step(*a)) or steps[-1]
    return steps


def log_softmax(x):
    x = x.astype(np.float64)
    m = x.max(-1, keepdims=True)
    return x - m - np.log(np.exp(x - m).sum(-1, keepdims=True))


def replay(prompt_logits, steps, beams, eos):
    """A request's search over the logits that the decoder saw: (tokens, score) of its beams in their order. A beam that has
    ended keeps its place at its own score."""
    lp = log_softmax(prompt_logits)
    best = np.argsort(-lp, kind="stable")[:beams]
    alive = [([int(t)], float(np.float32(lp[t]))) for t in best]
    for logits in steps:
        lp, cand = log_softmax(logits), []
        for k, (tokens, s) in enumerate(alive):
            if tokens[-1] == eos:
                cand.append((s, k, None))
            else:
                cand += [(s + lp[k, t], k, int(t)) for t in np.argsort(-lp[k], kind="stable")[:beams]]
        cand.sort(key=lambda c: -c[0])
        alive = [(alive[k][0] + ([t] if t is not None else []), float(np.float32(s))) for s, k, t in cand[:beams]]
    return alive


@pytest.mark.parametrize("bits, page", [(16, 4), (16, 16), (8, 4), (16, 1)])
def test_hypotheses_that_end_keep_their_score_and_tokens(bits, page):
    """Beams that have ended stay beside the others at their own score, are followed by longer ones and follow shorter ones;
    histories, lengths and scores are those of the same search on the host, over the decoder's own logits."""
    cfg, params, prompts, d = make_ending(bits, page)
    steps = recorded(d)
    out = d.search()
    assert len(steps) == 8  # (one request's beams never end)
    host = [s.cpu().numpy() for s in steps]
    ends = set()
    for g, beams in enumerate(out):
        want = replay(d.prompt_logits[g].cpu().numpy(), [s[g] for s in host], 4, cfg.eos_id)
        assert [t for t, _ in beams] == [t for t, _ in want]
        # a step's log-sum-exp in fp32 (2^-20 relative to values of up to 32) and its rounding
        assert np.allclose([s for _, s in beams], [s for _, s in want], rtol=0, atol=9 * 2.0 ** -15)
        for tokens, _ in beams:
            ended = tokens[-1] == cfg.eos_id
            assert cfg.eos_id not in tokens[:-1] and (ended or len(tokens) == 9)
            ends.add(len(tokens) if ended else 0)
    assert 0 in ends and len(ends) >= 4  # some go on to the last step, others end at three different ones at least


def test_scores_of_ended_hypotheses_are_the_forward_pass_log_probabilities():
    """The decoder's and the context's logits are as far apart as test_gpu_beam_decode.TOL has it, times the final norm's factor
    of four and the end-of-sequence row's larger norm; a token's log-probability twice that."""
    from tests.test_gpu_beam_decode import TOL, score
    cfg, params, prompts, d = make_ending(16, 4)
    rows = np.linalg.norm(params[:cfg.vocab_size * cfg.d_model].reshape(cfg.vocab_size, -1), axis=1)
    tol = 2 * TOL["tiny"] * 4 * max(1.0, rows[cfg.eos_id] / np.median(rows))
    ex = E.make_execution(cfg, params)
    for prompt, beams in zip(prompts, d.search()):
        for tokens, s in beams:
            assert abs(s - score(ex, prompt, tokens)) <= tol * len(tokens)


def test_a_search_stops_where_all_hypotheses_have_ended():
    """A request whose beams end early: no step is made after the last one has ended, and a second search is the same."""
    cfg, _, _, d = make_ending(16, 4, lens=(1,), new=40, share=0.8)
    steps = recorded(d)
    out = d.search()
    longest = max(len(t) for t, _ in out[0])
    assert all(t[-1] == cfg.eos_id for t, _ in out[0]) and len(steps) == longest - 1 < 39
    assert [t for t, _ in out[0]] == [t for t, _ in replay(d.prompt_logits[0].cpu().numpy(), [s[0].cpu().numpy() for s in steps], 4, cfg.eos_id)]
    assert d.search() == out


def test_length_penalty_reorders_hypotheses_of_different_lengths():
    _, _, _, d = make_ending(16, 4)
    plain, means = d.search(), d.search(length_penalty=1.0)
    for a, b in zip(plain, means):
        assert sorted(a) == sorted(b)
        assert [x[0] for x in b] == [x[0] for x in sorted(a, key=lambda x: -x[1] / len(x[0]))]
    assert [[t for t, _ in b] for b in plain] != [[t for t, _ in b] for b in means]


# ------------------------------------------------------------------ a window over the prompt
def windowed_logits(cfg, params, ids, window, sinks):
    """The model in 64 bits, in which token t sees the last `window` tokens up to itself and the first `sinks`: logits [T, V]."""
    from oracle import mla_oracle as O
    P = O.Params(cfg, [t.astype(np.float64) for t in O.split_params(cfg, params)])
    T, H, N, R, L = len(ids), cfg.n_heads, cfg.head_dim_nope, cfg.head_dim_rope, cfg.kv_lora_rank
    norm = lambda x, w: x / np.sqrt((x * x).mean(-1, keepdims=True) + cfg.norm_epsilon) * w.reshape(-1)  # noqa: E731
    angle = np.arange(T)[:, None] * cfg.rope_theta ** (-np.arange(0, R, 2) / R)

    def turn(x):  # [T, ..., R]
        a, b = x[..., 0::2], x[..., 1::2]
        shape = (T,) + (1,) * (x.ndim - 2) + (R // 2,)
        c, s = np.cos(angle).reshape(shape), np.sin(angle).reshape(shape)
        return np.stack([a * c - b * s, a * s + b * c], -1).reshape(x.shape)

    t, j = np.arange(T)[:, None], np.arange(T)[None]
    seen = (j <= t) & ((j > t - window) | (j < sinks))
    x = P.embedding[np.asarray(ids)]
    for l in range(cfg.n_layers):
        w = lambda n: P.layer(l, n)  # noqa: B023, E731
        h = norm(x, w("attn_norm"))
        q = (norm(h @ w("w_dq"), w("q_norm")) @ w("w_uq")).reshape(T, H, N + R)
        kv = h @ w("w_dkv")
        latent, rope = norm(kv[:, :L], w("kv_norm")), turn(kv[:, L:])
        s = np.einsum("thn,jhn->htj", q[..., :N], (latent @ w("w_uk")).reshape(T, H, N)) + np.einsum("thr,jr->htj", turn(q[..., N:]), rope)
        s = np.where(seen, s / np.sqrt(N + R), -np.inf)
        p = np.exp(s - s.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        o = np.einsum("htj,jhv->thv", p, (latent @ w("w_uv")).reshape(T, H, -1)).reshape(T, -1)
        x = x + o @ w("w_o")
        h = norm(x, w("ffn_norm"))
        gate = h @ w("w_gate")
        x = x + (gate / (1 + np.exp(-gate)) * (h @ w("w_up"))) @ w("w_down")
    return norm(x, P.final_norm) @ P.embedding.T


@pytest.mark.parametrize("name", ["tiny", "mla36m"])
@pytest.mark.parametrize("window, sinks", [(3, 1), (1, 0)])
def test_a_windowed_search_is_the_windowed_model(name, window, sinks):
    """Prompt logits and every hypothesis' score against the 64-bit model, within what test_gpu_beam_decode.TOL allows the
    logits; without the window they are further apart than that."""
    from tests.test_gpu_beam_decode import TOL
    cfg, params, prompts, d = make(name, window=window, sinks=sinks)
    for g, prompt in enumerate(prompts):
        got = d.prompt_logits[g].double().cpu().numpy()
        assert np.abs(got - windowed_logits(cfg, params, prompt, window, sinks)[-1]).max() <= TOL[name]
    for prompt, beams in zip(prompts, d.search()):
        for tokens, s in beams:
            lp = log_softmax(windowed_logits(cfg, params, prompt + tokens[:-1], window, sinks))[len(prompt) - 1:]
            assert abs(s - sum(lp[i, t] for i, t in enumerate(tokens))) <= 2 * TOL[name] * len(tokens)
    long = prompts[0]
    apart = windowed_logits(cfg, params, long, window, sinks) - windowed_logits(cfg, params, long, len(long), 0)
    assert np.abs(apart[-1]).max() > 3 * TOL[name]
