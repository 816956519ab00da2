"""Group decode with shared prompts and drafted tokens (group_decode.py) against the context's own
forward pass."""
import numpy as np
import pytest

import cpp_inference_train_engine_b200 as E
from cpp_inference_train_engine_b200.config import MLA36M, TINY
from tests.gpu_util import require_gpu

pytestmark = pytest.mark.gpu

# both sides' fp16 logits are held to these against the fp32 decoder (test_gpu_decode.py): twice that apart
TOL = {"tiny": 2 * 5e-3, "mla36m": 2 * 2e-2}
CONFIGS = {"tiny": TINY, "mla36m": MLA36M}


def make(name, bits, new=12, drafts=3, rows=(3, 1, 2), lens=(17, 1, 9)):
    require_gpu()
    from cpp_inference_train_engine_b200.group_decode import GroupDecoder
    cfg = CONFIGS[name]
    params = E.init_params(cfg, 3)
    rng = np.random.default_rng(4)
    prompts = [rng.integers(0, 256, n).tolist() for n in lens]
    return cfg, params, prompts, GroupDecoder(cfg, params, prompts, list(rows), new, drafts, bits)


@pytest.mark.parametrize("name", CONFIGS)
def test_logits_match_the_context_forward(name):
    """Prompt logits, then steps of several tokens and of one over the shared prompts."""
    import torch
    cfg, params, prompts, d = make(name, 16)
    ex = E.make_execution(cfg, params)
    for i, p in enumerate(prompts):
        want = ex.forward(np.array(p), 1, len(p))[-1]
        assert np.abs(d.prompt_logits[i].cpu().numpy() - want).max() < TOL[name]
    rng = np.random.default_rng(5)
    groups = d.row_group.tolist()
    chosen = rng.integers(0, 256, (len(groups), 7))
    at = 0
    for T in (3, 1, 2):
        tokens = torch.tensor(chosen[:, at:at + T], dtype=torch.int32, device="cuda")
        d._append(tokens[:, :1], torch.ones_like(d.count))  # the last token a row has; the others are drafts
        got = d.step_logits(tokens).cpu().numpy()
        for b, g in enumerate(groups):
            ids = np.array(prompts[g] + chosen[b, :at + T].tolist())
            want = ex.forward(ids, 1, len(ids))[-T:]
            assert np.abs(got[b] - want).max() < TOL[name], (T, b)
        if T > 1:  # all accepted
            d._append(tokens[:, 1:], torch.full_like(d.count, T - 1))
        at += T


@pytest.mark.parametrize("name", CONFIGS)
@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("drafts", [0, 3])
def test_greedy_completions_follow_the_forward_pass(name, bits, drafts):
    """Each greedy token is the argmax (to the tolerance) of a plain one-token replay."""
    import torch
    cfg, params, prompts, d = make(name, bits, drafts=drafts)
    out, stats = d.generate()
    assert stats["accepted"] <= stats["proposed"] and stats["tokens"] == sum(map(len, out))
    assert all(1 <= len(o) <= 12 and (len(o) == 12 or o[-1] == cfg.eos_id) for o in out)
    assert all(cfg.eos_id not in o[:-1] for o in out)
    groups = d.row_group.tolist()
    if bits == 16:
        ex = E.make_execution(cfg, params)
        for b, o in enumerate(out):
            p = prompts[groups[b]]
            lg = ex.forward(np.array(p + o[:-1]), 1, len(p) + len(o) - 1)[len(p) - 1:]
            for i, t in enumerate(o):
                assert lg[i, t] >= lg[i].max() - 2 * TOL[name], (b, i)
        return
    r = make(name, bits, drafts=0)[3]
    logits = r.prompt_logits[r.row_group]
    for i in range(12):
        forced = torch.tensor([[o[i]] if i < len(o) else [0] for o in out], dtype=torch.int32, device="cuda")
        for b, o in enumerate(out):
            if i < len(o):
                assert logits[b, o[i]] >= logits[b].max() - 2 * TOL[name], (b, i)
        r._append(forced, torch.ones_like(r.count))
        logits = r.step_logits(forced)[:, 0]


def test_stored_prompt_rows_keep_their_values():
    """The first layer's 8-bit prompt rows read back within an e4m3 rounding of the 16-bit ones."""
    import torch
    a, b = make("mla36m", 16)[3], make("mla36m", 8)[3]
    for g in range(3):
        x, y = a.stored(0, g).double(), b.stored(0, g).double()
        assert x.shape == y.shape and torch.equal(x[:, 128:], y[:, 128:])
        lat, amax = x[:, :128], x[:, :128].abs().amax(1, keepdim=True)
        # four significant bits, steps of 2^-9 scales below the normal range, and fp16 roundings of both
        assert torch.all((lat - y[:, :128]).abs() <= lat.abs() * (2.0 ** -4 + 2.0 ** -9) + amax / 448 * 2.0 ** -10)
    assert b.cache_bytes() < 0.65 * a.cache_bytes()


def test_sampling_depends_on_the_seed_alone():
    a = make("tiny", 8)[3].generate(1.0, 7)[0]
    assert a == make("tiny", 8)[3].generate(1.0, 7)[0]
    assert a != make("tiny", 8)[3].generate(1.0, 8)[0]


def test_command_reports_its_work(capsys):
    require_gpu()
    from cpp_inference_train_engine_b200 import group_decode
    group_decode.main(["--model", "tiny", "--groups", "2", "--rows", "3", "--prompt", "9", "--new", "5", "--drafts", "2"])
    assert "tokens/s" in capsys.readouterr().out
