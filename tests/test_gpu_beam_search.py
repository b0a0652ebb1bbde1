"""Whole beam searches on the GPU: attention with first tokens, the choice of beams and the moving of their states together, against a
plain search over the oracle in 64 bits; beside other requests, from CUDA graphs, through the engine and the command line."""
import pytest
import torch

from oracle import hybrid_oracle as O
from tests import hybrid_util as U
from tests.beam_util import plain_search

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def exact_products():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    torch.set_float32_matmul_precision("highest")


def first(m, n):
    m["mask"]["first"] = n
    return m


# every kind of state that follows a beam; windows that a prompt and a few tokens fill and pass, with and without first tokens
MODELS = {
    "parallel": U.parallel(64, 61, [
        U.layer("wkv", U.wkv(2, 24), U.dense(48)),
        U.layer("attention", first(U.attention(4, 2, 16, 12, 7, 8, 3), 2), U.dense(40)),
        U.layer("mamba2", U.mamba2(4, 8, 12, 2, 2, 4), None),
        U.layer("attention", U.attention(2, 1, 16, 16, None, 8, 1), U.dense(32)),
    ], loop={"start": 1, "stop": 3, "times": 2}, bigram=(31, 7, 3), cap=12.0),
    "sandwich": U.config(64, 53, [
        U.layer("delta", U.delta(4, 2, 16, 12, 4), U.dense(48)),
        U.layer("latent_attention", U.latent(3, 16, 8, 12, 24, 9), None),
        U.layer("attention", first(U.attention(3, 3, 9, 5, 5, 4, 2), 11), U.dense(21)),
    ]),
}
_MADE = {}


def made(name):
    from msa_b200.hybrid import HybridForCausalLM
    from msa_b200.hybrid_config import HybridConfig
    if name not in _MADE:
        w = U.make_weights(MODELS[name], 11)
        _MADE[name] = w, HybridForCausalLM(HybridConfig.parse(MODELS[name]), w, "cuda:0", torch.float32)
    return _MADE[name]


_LOG_PROBS = {}


def wanted(name, prompt, beams, n, stop=(), penalty=1.0):
    """The plain search; a search whose outcome hangs on differences that fp32 does not resolve would not do as a test."""
    w, _ = made(name)

    def log_probs(toks):
        key = (name, tuple(prompt) + tuple(toks))
        if key not in _LOG_PROBS:
            _LOG_PROBS[key] = torch.log_softmax(O.forward(MODELS[name], w, list(key[1]))[-1], 0)
        return _LOG_PROBS[key]
    return plain_search(log_probs, beams, n, stop, penalty)


def same(request, want):
    assert [t for _, t in request.results] == [t for _, t in want]
    assert all(abs(a - b) < 1e-3 for (a, _), (b, _) in zip(request.results, want)) and request.output == want[0][1]


@pytest.mark.parametrize("graphs", [False, True], ids=["steps", "graphs"])
@pytest.mark.parametrize("name", list(MODELS))
def test_searches_beside_other_requests(name, graphs):
    from msa_b200.scheduler import Scheduler, SequenceRequest
    _, m = made(name)
    vocab = MODELS[name]["vocab"]
    s = Scheduler(m, max_batch=10, max_len=32, portion=6, step_tokens=16, graphs=graphs)
    reqs = [SequenceRequest(U.tokens_of(MODELS[name], n, 40 + i), k, beams=b, eos_token_ids=stop, length_penalty=p)
            for i, (n, k, b, stop, p) in enumerate([(9, 8, 4, [], 1.0), (4, 8, 1, [], 1.0), (13, 7, 4, [vocab - 1, 3], 0.5), (2, 8, 3, [5], 1.0), (1, 6, 2, [], 1.0),
                                                    (17, 6, 6, [7], 0.0)])]
    for r in reqs:
        s.submit(r)
    assert len(s.run()) == len(reqs) and s.cache.free_slots == 10
    for r in reqs:
        want = wanted(name, r.tokens, r.beams, r.max_new_tokens, r.eos_token_ids, r.length_penalty)
        if r.beams > 1:
            same(r, want)
        else:
            assert r.output == want[0][1]
    if graphs:
        assert s._graphs


def test_a_wide_search():
    """32 beams: what comes out is a search's result, ratings in order and sums of the model's own log probabilities."""
    from msa_b200.scheduler import Scheduler, SequenceRequest
    cfg, m = MODELS["parallel"], made("parallel")[1]
    s = Scheduler(m, max_batch=32, max_len=32)
    r = SequenceRequest(U.tokens_of(cfg, 7, 3), 9, beams=32, eos_token_ids=[2])
    s.submit(r)
    s.run()
    assert len(r.results) == 32 and [a for a, _ in r.results] == sorted((a for a, _ in r.results), reverse=True) and len({tuple(t) for _, t in r.results}) == 32
    cache = m.new_cache(1, 32)
    for rating, toks in r.results[::5]:
        cache.acquire("x")
        logits = m.run([("x", r.tokens + toks[:-1], list(range(6, 6 + len(toks))))], cache)
        cache.release("x")
        lp = torch.log_softmax(logits.double(), 1).cpu()
        got = sum(float(lp[i, t]) for i, t in enumerate(toks)) / len(toks)
        # single tokens there, one portion here: rows of logits (of size 3) within 2e-4 of the oracle each, twice that in a log probability
        assert abs(got - rating) < 2.4e-3, (got, rating)


@pytest.mark.timeout(300)
def test_engine_and_command_line_search(tmp_path, capfd):
    from msa_b200.__main__ import main
    from msa_b200.engine import GenerateConfig, MSAEngine
    from msa_b200.memory import ModelConfig
    name = "parallel"
    cfg = MODELS[name]
    U.save(cfg, made(name)[0], str(tmp_path))
    prompts = [U.tokens_of(cfg, n, 80 + n) for n in (12, 3)]
    want = [" ".join(map(str, wanted(name, p, 3, 5)[0][1])) for p in prompts]
    gen = GenerateConfig(devices=[0], max_generate_tokens=5, max_context=64, state_slots=4, num_beams=3)
    with MSAEngine(gen, ModelConfig(model_path=str(tmp_path), dtype="float32")) as e:
        assert e.generate(prompts)[0] == want
    assert main(["generate", "--model", str(tmp_path), "--tokens", ",".join(map(str, prompts[0])), "--max-new-tokens", "5", "--beams", "3",
                 "--max-context", "64", "--dtype", "float32"]) == 0
    assert want[0] in capfd.readouterr().out
