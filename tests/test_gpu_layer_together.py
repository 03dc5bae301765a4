"""A layer of linear attention as a model uses its operators: projections, head norms with the rotary
embedding, attention with decays, the logits and the scores of the tokens; trained, and answering token by
token from a prompt's state.

Tolerances: float32 matrix products of the layer have 64 to 300 terms, and four of them, the attention and the
scores follow one another, so that fewer than 2048 roundings of 2^-24 meet in a result."""

import pytest
import torch

from oal_amd.decay_attention import decay_attention, decay_step
from oal_amd.norm_rotary import norm_rotary_heads
from oal_amd.token_scores import token_log_probs
from oracle.decay_oracle import decay_attention as exact_attention
from oracle.heads_oracle import norm_rotary, token_scores

pytestmark = pytest.mark.gpu

_HQ, _HK, _D, _WIDTH, _VOCAB = 6, 2, 32, 96, 301
_TOL = 2048 * 2.0 ** -24


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda:0")


def _model(dtype=torch.float32):
    gen = torch.Generator().manual_seed(3)

    def normal(*shape):
        return torch.randn(*shape, generator=gen)

    sizes = dict(embed=(_VOCAB, _WIDTH), qkv=((_HQ + 2 * _HK) * _D, _WIDTH), out=(_WIDTH, _HQ * _D), gate=(_HK, _WIDTH))
    weights = {name: (normal(*shape) * shape[1] ** -0.5).to(dtype) for name, shape in sizes.items()}
    weights["q_norm"], weights["k_norm"] = 1 + 0.1 * normal(_D), 1 + 0.1 * normal(_D)
    angle = torch.outer(torch.arange(400, dtype=torch.float64), 1e4 ** (-torch.arange(0, _D, 2, dtype=torch.float64) / _D))
    return weights, angle.repeat(1, 2).cos().float(), angle.repeat(1, 2).sin().float()


def _hidden(w, tokens):
    return torch.nn.functional.embedding(tokens, w["embed"])


def _split(w, x):
    return torch.nn.functional.linear(x, w["qkv"]).split([_HQ * _D, _HK * _D, _HK * _D], -1)


def _gates(w, x):
    """A decay for each token and KV head."""
    return torch.nn.functional.logsigmoid(torch.nn.functional.linear(x, w["gate"]).float()).transpose(1, 2)


def _logits(w, x, o):
    x = x + torch.nn.functional.linear(o.transpose(1, 2).flatten(2), w["out"])
    return torch.nn.functional.linear(x, w["embed"])


def _forward(w, cos, sin, tokens, attention, heads, state=None, positions=None):
    x = _hidden(w, tokens)
    q, k, v = heads(*_split(w, x), w["q_norm"], w["k_norm"], cos, sin, q_heads=_HQ, kv_heads=_HK, eps=1e-6, positions=positions)
    return x, attention(q, k, v, _gates(w, x), state)


def _mine(q, k, v, g, state):
    return decay_attention(q, k, v, g, initial_state=state)


def _exact(q, k, v, g, state):
    return exact_attention(q, k, v, g.double(), state, scale=_D ** -0.5)


def test_training():
    dev = _dev()
    weights, cos, sin = _model()
    tokens = torch.randint(0, _VOCAB, (2, 150), generator=torch.Generator().manual_seed(5))
    w = {name: t.double().requires_grad_() for name, t in weights.items()}
    x = _hidden(w, tokens)
    q, k, v = norm_rotary(*_split(w, x), w["q_norm"], w["k_norm"], cos, sin, q_heads=_HQ, kv_heads=_HK, eps=1e-6)
    gates = torch.nn.functional.logsigmoid(torch.nn.functional.linear(x, w["gate"])).transpose(1, 2)
    o, _ = exact_attention(q, k, v, gates, scale=_D ** -0.5)
    log, entropy = token_scores(_logits(w, x, o)[:, :-1], tokens[:, 1:])
    want = [log, entropy, *torch.autograd.grad(0.01 * entropy.mean() - log.mean(), list(w.values()))]

    w = {name: t.to(dev).requires_grad_() for name, t in weights.items()}
    x, (o, _) = _forward(w, cos.to(dev), sin.to(dev), tokens.to(dev), _mine, norm_rotary_heads)
    scores = token_log_probs(_logits(w, x, o)[:, :-1], tokens[:, 1:].to(dev), entropy=True)
    got = [*scores[:2], *torch.autograd.grad(0.01 * scores.entropy.mean() - scores.log_probs.mean(), list(w.values()))]
    for name, a, b in zip(["log_probs", "entropy", *w], got, want):
        a, b = a.detach().cpu().double(), b.detach()
        assert float((a - b).norm()) <= _TOL * float(b.norm()), name


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_answering_token_by_token(dtype):
    """Prompts of two lengths in one padded batch, then tokens one at a time, in a captured step: the scores are
    those of the whole texts."""
    dev = _dev()
    weights, cos, sin = _model(dtype)
    w = {name: t.to(dev) for name, t in weights.items()}
    cos, sin = cos.to(dev), sin.to(dev)
    total, lengths = 90, torch.tensor([70, 41], device=dev)
    tokens = torch.randint(0, _VOCAB, (2, total), generator=torch.Generator().manual_seed(7)).to(dev)
    with torch.no_grad():
        x, (o, _) = _forward(w, cos, sin, tokens, _mine, norm_rotary_heads)
        whole = token_log_probs(_logits(w, x, o)[:, :-1], tokens[:, 1:], entropy=True, top=3)
        # the prompts: behind its end a sequence has no tokens
        at = torch.arange(70, device=dev).expand(2, 70)
        there = at < lengths[:, None]
        x = _hidden(w, tokens[:, :70])
        q, k, v = norm_rotary_heads(*_split(w, x), w["q_norm"], w["k_norm"], cos, sin, q_heads=_HQ, kv_heads=_HK,
                                    positions=torch.where(there, at, -1))
        _, state = decay_attention(q, k, v, torch.where(there[:, None], _gates(w, x), 0.0))

        token, position = tokens[:, :1].clone(), lengths[:, None].clone()
        target = tokens[:, :1].clone()
        rows = torch.arange(2, device=dev)[:, None]

        def step():
            x = _hidden(w, token)
            q, k, v = norm_rotary_heads(*_split(w, x), w["q_norm"], w["k_norm"], cos, sin, q_heads=_HQ, kv_heads=_HK,
                                        positions=position)
            o = decay_step(q, k, v, _gates(w, x), state)
            return token_log_probs(_logits(w, x, o), target, entropy=True, top=3)

        start = state.clone()
        side = torch.cuda.Stream(dev)
        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream(dev).wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step()
        state.copy_(start)
        # bf16: every value of the residual and of the logits is rounded, each by at most 2^-8, in sums of up to 300 terms
        tol = _TOL if dtype is torch.float32 else 8 * 2.0 ** -8
        for n in range(15):
            position.copy_(lengths[:, None] + n)
            token.copy_(tokens[rows, position])
            target.copy_(tokens[rows, position + 1])
            graph.replay()
            for name, got, want in zip(held._fields, held, whole):
                want = want[rows, position]
                if name == "top_tokens":
                    assert dtype is torch.bfloat16 or torch.equal(got, want)
                else:
                    assert float((got - want).norm()) <= tol * float(want.norm()), (name, n)


def test_the_model_scores_its_tokens():
    from oal_amd.qwen_oal import QwenOALConfig, QwenOALModel, score_tokens

    dev = _dev()
    cfg = QwenOALConfig(vocab_size=501, hidden_size=128, intermediate_size=256, num_layers=2, num_heads=4, num_kv_heads=2,
                        lora_rank=4)
    model = QwenOALModel(cfg, seed=1).to(dev).cast_parameters_(torch.bfloat16)
    tokens = torch.randint(0, 501, (2, 77), generator=torch.Generator().manual_seed(9)).to(dev)
    scores = score_tokens(model, tokens, entropy=True, top=5)
    with torch.no_grad():
        logits = model(tokens)
    log, entropy = token_scores(logits[:, :-1], tokens[:, 1:])
    for got, want in ((scores.log_probs, log), (scores.entropy, entropy)):
        assert got.shape == (2, 76) and float((got.double() - want).norm()) <= 200 * 2.0 ** -24 * float(want.norm())
    assert scores.top_tokens.shape == (2, 76, 5) and not scores.log_probs.requires_grad
    # what a padded batch's places are worth counts for nothing
    short = score_tokens(model, tokens, lengths=torch.tensor([77, 30], device=dev))
    assert torch.equal(short.log_probs[0], scores.log_probs[0]) and torch.equal(short.log_probs[1, :29], scores.log_probs[1, :29])
    assert not short.log_probs[1, 29:].any() and short.entropy is None
