"""Sampling on the GPU against the sorted 64-bit form: equal tokens, and probabilities within f32 rounding.

The kernel's weights are integers of 2^-40 of the largest weight or finer, the oracle's 64-bit floats: a token could differ only where
u times the kept weight lies within about 1e-9 of a running sum, which 24-bit random numbers over these rows meet with a chance below 1e-5
for a whole run; exact ties (equal logits) are exact in both."""
import numpy as np
import pytest

from tests.serve_oracle import draw

pytestmark = pytest.mark.gpu


def _draw(lg, logits, u, guard=None, **params):
    """(tokens, probs) through the GPU; params: a number for all rows or one a row; guard: columns of junk behind each row."""
    import torch
    rows = len(u)
    kinds = {"temperature": np.float32, "top_k": np.int32, "top_p": np.float32, "min_p": np.float32}
    dev = {k: torch.tensor(np.broadcast_to(np.asarray(v, dtype=kinds[k]), rows).copy(), device="cuda") for k, v in params.items() if v is not None}
    token = torch.full((rows + 1,), -9, dtype=torch.int32, device="cuda")
    prob = torch.full((rows + 1,), -9.0, device="cuda")
    lg.sample(logits, torch.tensor(np.asarray(u, np.float32), device="cuda"), token, prob, **dev)
    token, prob = token.cpu().numpy(), prob.cpu().numpy()
    assert token[rows] == -9 and prob[rows] == -9.0
    return token[:rows], prob[:rows]


def _check(lg, logits, u, **params):
    token, prob = _draw(lg, logits, u, **params)
    host = logits.double().cpu().numpy()
    for r in range(len(u)):
        one = {k: float(np.asarray(np.broadcast_to(v, len(u))[r], np.float32)) if k != "top_k" else int(np.broadcast_to(v, len(u))[r]) for k, v in params.items() if v is not None}
        want, p = draw(host[r], float(np.float32(u[r])), **one)
        assert token[r] == want, (r, one, u[r], token[r], want, prob[r], p)
        # rounding to f32, and the integer sum it is divided by (2^-24 of the largest weight at most)
        assert abs(prob[r] - p) <= 2.0 ** -22 * p + 1e-30, (r, one, prob[r], p)
    return token, prob


def _logits(rows, vocab, dtype="float32", seed=0, spread=2.0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((rows, vocab), generator=g, device="cuda") * spread
    x += torch.where(torch.rand((rows, vocab), generator=g, device="cuda") < 12.0 / vocab, 7.0, 0.0)
    return x.to(getattr(torch, dtype))


FILTERS = [dict(), dict(temperature=0.7), dict(top_k=1), dict(top_k=50), dict(top_k=50, top_p=0.9), dict(top_p=0.5), dict(top_p=0.95, min_p=0.02), dict(min_p=0.1),
           dict(temperature=1.4, top_k=900, top_p=0.99, min_p=0.001)]


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("vocab", [1, 2, 31, 33, 1000, 4097, 32768, 50257, 262144, 300001])
def test_draws_equal_the_sorted_form(lg, dtype, vocab):
    rng = np.random.default_rng(vocab)
    for i, f in enumerate(FILTERS):
        rows = 7 if vocab < 100000 else 3
        _check(lg, _logits(rows, vocab, dtype, seed=i), rng.random(rows, dtype=np.float32), **f)


@pytest.mark.parametrize("rows", [1, 2, 9, 150, 600])
def test_every_row_has_parameters_of_its_own(lg, rows):
    rng = np.random.default_rng(rows)
    _check(lg, _logits(rows, 3001, seed=rows), rng.random(rows, dtype=np.float32), temperature=rng.choice([0.0, 0.3, 1.0, 2.5, -1.0], rows),
           top_k=rng.choice([0, -3, 1, 7, 3000, 3001, 1 << 30], rows), top_p=rng.choice([0.0, 0.2, 0.9, 1.0, 1.5], rows), min_p=rng.choice([0.0, 0.05, 1.0, 1.5], rows))


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_ties_go_to_the_lowest_index(lg, dtype):
    """Rows of few different logits, where filters cut through groups of equals."""
    import torch
    rng = np.random.default_rng(1)
    for vocab in (40, 5000, 140001):
        x = torch.tensor(rng.integers(-2, 3, (4, vocab)) * 0.5, device="cuda").to(getattr(torch, dtype))
        for f in (dict(top_k=7), dict(top_k=vocab // 2), dict(top_p=0.5), dict(top_k=vocab // 2 + 1, top_p=0.7), dict(top_p=0.25, min_p=0.3), dict(temperature=0.0), dict(top_p=1e-6)):
            _check(lg, x, rng.random(4, dtype=np.float32), **f)
    x = torch.zeros((3, 1000), device="cuda").to(getattr(torch, dtype))
    x[:, ::2] = -0.0                                                             # -0 is 0
    token, prob = _check(lg, x, [0.0, 0.5, 0.999], top_k=10)
    assert token.tolist() == [0, 5, 9] and np.allclose(prob, 0.1)
    token, _ = _check(lg, x, [0.0, 0.4999, 0.5], top_p=0.5)                       # 500 of 1000 equals, exactly
    assert token.tolist() == [0, 249, 250]


@pytest.mark.parametrize("dtype,vocab", [("float32", 262144), ("bfloat16", 262144), ("float32", 1000000), ("float16", 20000)])
@pytest.mark.parametrize("spread", [1e-4, 0.05, 1.0])
def test_flat_rows(lg, dtype, vocab, spread):
    """Hundreds of thousands of tokens near a threshold: more than lists and single CTAs hold."""
    rng = np.random.default_rng(vocab)
    rows = 3
    x = _logits(rows, vocab, dtype, seed=vocab, spread=spread)
    x[:, ::7] = x[:, :1]
    for f in (dict(top_p=0.5), dict(top_k=vocab // 3, top_p=0.7), dict(top_k=1500, top_p=0.9), dict(top_k=2049), dict(top_p=0.99, min_p=0.4), dict(temperature=5.0, top_p=0.3)):
        _check(lg, x, rng.random(rows, dtype=np.float32), **f)


@pytest.mark.parametrize("rows,vocab", [(40, 100000), (200, 33000), (90, 262144)])
def test_rows_shared_by_other_numbers_of_ctas(lg, rows, vocab):
    rng = np.random.default_rng(rows)
    x = _logits(rows, vocab, "bfloat16", seed=rows)
    for f in (dict(top_p=0.9), dict(top_k=60, top_p=0.8, min_p=0.05)):
        _check(lg, x, rng.random(rows, dtype=np.float32), temperature=rng.choice([0.5, 1.0, 1.5, 0.0], rows), **f)


def test_ruled_out_tokens_and_empty_rows(lg):
    import torch
    inf = float("inf")
    x = _logits(8, 5000)
    x[0] = -inf
    x[1] = float("nan")
    x[2, :] = -inf; x[2, 4321] = -3e38                                            # one token left
    x[3, ::2] = float("nan"); x[3, 1::4] = -inf
    x[4, 17] = inf; x[4, 4000] = inf; x[4, 3] = float("nan")
    x[5] = torch.finfo(torch.float32).min                                         # the type's lowest value everywhere: no mask, all equal
    x[6, 100:] = torch.finfo(torch.float32).min
    for f in FILTERS:
        token, prob = _check(lg, x, [0.3, 0.3, 0.9, 0.6, 0.7, 0.5, 0.99, 0.1], **f)
        assert token[0] == token[1] == -1 and prob[0] == prob[1] == 0.0 and token[2] == 4321 and prob[2] == 1.0 and token[4] in (17, 4000)


def test_random_numbers_at_and_outside_of_their_range(lg):
    x = _logits(6, 3333)
    u = np.array([0.0, 1.0 - 2.0 ** -24, 1.0, 7.0, -1.0, np.nan], np.float32)
    token, _ = _draw(lg, x, u, top_k=20)
    kept = [np.sort(np.lexsort((np.arange(3333), -r))[:20]) for r in x.double().cpu().numpy()]
    assert [int(t) for t in token] == [int(k[i]) for k, i in zip(kept, (0, -1, -1, -1, 0, 0))]


def test_temperatures_at_the_ends(lg):
    x = _logits(5, 2000, seed=3)
    _check(lg, x, [0.5] * 5, temperature=np.array([1e-30, 1e-45, 1e30, np.inf, 0.01], np.float32))
    token, prob = _draw(lg, x, [0.5] * 5, temperature=np.nan)
    assert token.tolist() == x.argmax(-1).tolist() and (prob == 1.0).all()


@pytest.mark.parametrize("dtype,ld,shift", [("float32", 1001, 1), ("bfloat16", 1003, 3), ("float16", 1024, 5)])
def test_rows_apart_and_at_odd_addresses(lg, dtype, ld, shift):
    import torch
    flat = torch.full((6 * ld + 8,), float("inf"), device="cuda").to(getattr(torch, dtype))     # what lies between rows would win
    x = flat[shift:shift + 6 * ld].view(6, ld)[:, :999]
    x.copy_(_logits(6, 999, dtype))
    for f in FILTERS:
        _check(lg, x, np.linspace(0, 0.99, 6), **f)


def test_shares_of_draws(lg):
    """Over evenly spread random numbers the tokens come as often as their probabilities say, to one part in the number of draws a token."""
    x = _logits(1, 500, seed=5).expand(2000, 500).contiguous()
    u = (np.arange(2000) + 0.5) / 2000
    token, prob = _draw(lg, x, u, top_k=30, top_p=0.9)
    for t in np.unique(token):
        assert abs((token == t).mean() - prob[token == t][0]) <= 1.0 / 2000


def test_no_rows_and_no_probabilities(lg):
    import torch
    token = torch.full((3,), -9, dtype=torch.int32, device="cuda")
    x = _logits(3, 100)
    lg.sample(x[:0], torch.zeros(0, device="cuda"), token)
    assert token.tolist() == [-9] * 3
    lg.sample(x, torch.zeros(3, device="cuda"), token, temperature=torch.zeros(3, device="cuda"))
    assert token.tolist() == x.argmax(-1).tolist()


def test_captured_on_a_stream_of_its_own(lg):
    import torch
    x, u = _logits(5, 40000), torch.rand(5, device="cuda")
    token, prob = torch.empty(5, dtype=torch.int32, device="cuda"), torch.empty(5, device="cuda")
    top_p = torch.full((5,), 0.8, device="cuda")
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        lg.sample(x, u, token, prob, top_p=top_p, stream=torch.cuda.current_stream().cuda_stream)
    for seed in range(3):
        x.copy_(_logits(5, 40000, seed=seed))
        u.uniform_()
        top_p.uniform_(0.1, 1.0)
        g.replay()
        torch.cuda.synchronize()
        for r in range(5):
            assert token[r].item() == draw(x[r].double().cpu().numpy(), u[r].item(), top_p=top_p[r].item())[0]


@pytest.mark.parametrize("name", ["tiny_cond"])
def test_session_draws_from_its_own_logits(lg, synth, name):
    from tests.conftest import model_files
    target, head = model_files(name)
    prompt = synth.prompt_ids(12, 4096, seed=2)
    with lg.Session(target, head, 128) as s:
        s.prefill(prompt[:-1], 0)
        logits = s.forward(int(prompt[-1]), 11)
        assert s.next_sampled(int(prompt[-1]), 11, 0.4, temperature=0.0) == (s.next(int(prompt[-1]), 11), 1.0)
        for u, f in ((0.1, dict()), (0.8, dict(temperature=0.7, top_k=40)), (0.99, dict(top_p=0.9, min_p=0.01)), (0.5, dict(top_k=1))):
            token, prob = s.next_sampled(int(prompt[-1]), 11, u, **f)
            want, p = draw(logits, float(np.float32(u)), **{k: v if k == "top_k" else float(np.float32(v)) for k, v in f.items()})
            assert token == want and abs(prob - p) <= 2.0 ** -22 * p
        # a sampled stream and a draft round on the same session
        token = int(prompt[-1])
        for pos in range(11, 20):
            token, _ = s.next_sampled(token, pos, 0.3, top_k=5)
        assert 0 <= token < s.n_vocab and s.next(token, 20) == s.forward(token, 20).argmax()


def test_session_of_a_layer_plan_draws_from_its_own_logits(lg):
    from tests.latent_models import model
    _, _, path = model("odd")
    with lg.Session(str(path), None, 64) as s:
        logits = s.forward(3, 0)
        token, prob = s.next_sampled(3, 0, 0.7, temperature=0.8, top_k=10)
        want, p = draw(logits, float(np.float32(0.7)), temperature=float(np.float32(0.8)), top_k=10)
        assert token == want and abs(prob - p) <= 2.0 ** -22 * p
