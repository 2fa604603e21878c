"""OlmoModel.generate_beam against a beam search in 64 bits that feeds every hypothesis from its beginning."""
import numpy as np
import pytest

from atlas_amd._lib import AtlasError, check, load
from tests import beam_ref, modelgen

pytestmark = pytest.mark.gpu

CONFIGS = {"olmo": dict(), "gqa": dict(n_kv_heads=1), "hd128": dict(n_heads=2, n_kv_heads=2),
           "pre-norm": dict(post_norm=False, qk_norm=False, yarn=None, n_kv_heads=2)}


def _weights(name, seed, fmt="bf16", **kw):
    return modelgen.make_weights(modelgen.olmo3_small_config(**CONFIGS[name], **kw), seed=seed, fmt=fmt)


def _prompt(seed, n):
    return np.random.default_rng(seed).integers(0, 512, n).tolist()


def _model(W, width, stops=(), **kw):
    m = modelgen.engine_model(W, max_batch=width, **kw)
    m.eos_token_id = stops[0] if stops else None
    m.extra_stop_tokens = list(stops[1:])
    return m


def _rescored(W, prompt, tokens, stop=None):
    ref = modelgen.Ref64(W)
    for t in prompt:
        z = ref.forward_one(int(t))
    total, seq = 0.0, list(tokens) + ([] if stop is None else [stop])
    for i, t in enumerate(seq):
        total += beam_ref.log_probs(z)[t]
        if i + 1 < len(seq):
            z = ref.forward_one(int(t))
    return total


# Scores: logits are within 1e-5 of each other at these sizes (activations in bf16 hi and lo, 2^-17, and f32 sums),
# so a sum of up to 30 log probabilities is within 1.5e-4.  Where every decision of the search has a larger gap,
# the hypotheses have to be the same.
TOL = 1.5e-4


@pytest.mark.parametrize("name,seed,width,max_new,penalty,n_prompt,stops", [
    ("olmo", 4, 6, 5, 0.0, 1, ()), ("olmo", 4, 6, 5, 0.0, 1, (303, 192)), ("olmo", 7, 4, 9, 1.0, 23, (72, 255)),
    ("gqa", 6, 6, 5, 0.0, 1, ()), ("gqa", 6, 6, 5, 0.0, 1, (235, 340)), ("olmo", 1, 1, 10, 1.0, 23, (126, 125))])
def test_beam_search_matches_64_bits(name, seed, width, max_new, penalty, n_prompt, stops):
    W, prompt = _weights(name, seed), _prompt(seed, n_prompt)
    want, gap = beam_ref.search(W, prompt, max_new, width, penalty, stops)
    assert gap > 2 * TOL
    got = _model(W, width, stops).generate_beam(prompt, max_new, width, penalty)
    assert [t for t, _ in got] == [t for t, _ in want]
    assert max(abs(a[1] - b[1]) for a, b in zip(got, want)) <= TOL


@pytest.mark.parametrize("name", list(CONFIGS))
@pytest.mark.parametrize("fmt,tol", [("bf16", TOL), ("int8", TOL), ("int4", 2e-2)])
@pytest.mark.parametrize("width,max_new,n_prompt", [(2, 30, 40), (16, 7, 3), (5, 20, 130)])
def test_beam_scores_are_their_tokens(name, fmt, tol, width, max_new, n_prompt):
    # (int4 products of activations keep 8 bits fewer)
    W, prompt = _weights(name, 11, fmt), _prompt(12, n_prompt)
    got = _model(W, width).generate_beam(prompt, max_new, width)
    assert len(got) == width and len({tuple(t) for t, _ in got}) == width
    assert [s for _, s in got] == sorted((s for _, s in got), reverse=True)
    for tokens, score in got[:3]:
        assert len(tokens) == max_new and abs(score - _rescored(W, prompt, tokens)) <= tol


def test_beam_search_of_one_is_greedy():
    W, prompt = _weights("olmo", 1), _prompt(1, 23)
    m = _model(W, 1)
    (tokens, _), = m.generate_beam(prompt, 10, 1)
    assert tokens == m.generate(prompt, 10, 0.0)


def test_beam_search_again_and_beside_other_calls():
    W, prompt = _weights("olmo", 5), _prompt(5, 33)
    m = _model(W, 8)
    greedy, batch = m.generate(prompt, 12, 0.0), m.generate_batch([prompt, prompt[:9]], 12)
    first = m.generate_beam(prompt, 25, 8)
    assert m.pos == 0
    other = m.generate_beam(prompt[:7], 9, 3)
    m.eos_token_id = other[0][0][2]
    stopped = m.generate_beam(prompt[:7], 9, 3)
    m.eos_token_id = None
    assert stopped != other and len(other) == 3
    assert m.generate(prompt, 12, 0.0) == greedy and m.generate_batch([prompt, prompt[:9]], 12) == batch
    assert m.generate_beam(prompt, 25, 8) == first and m.generate_beam(prompt[:7], 9, 3) == other
    assert _model(W, 8, use_graph=False).generate_beam(prompt, 25, 8) == first


def test_beam_search_to_the_end_of_the_cache():
    W = _weights("hd128", 3, max_seq=64)
    m, prompt = _model(W, 4), _prompt(3, 44)
    got = m.generate_beam(prompt, 20, 4)
    assert all(len(t) == 20 for t, _ in got) and abs(got[0][1] - _rescored(W, prompt, got[0][0])) <= TOL
    with pytest.raises(AtlasError):
        m.generate_beam(prompt, 21, 4)


def test_beam_search_nan_logits():
    W = _weights("olmo", 2)
    m = _model(W, 3)
    norm = np.full(256, np.nan, np.float32)
    m.set_tensor(13, 0, norm)          # the final norm's weights
    assert m.generate_beam([1, 2, 3], 5, 3) == []


def test_beam_search_refusals():
    W = _weights("olmo", 2)
    m = _model(W, 4)
    for args, code in (([[1, 2], 5, 0], -1), ([[1, 2], 5, 5], -1), ([[], 5, 2], -1), ([[1, 2], 0, 2], -1), ([[1, 2], 255, 2], -1),
                       ([[1, 2], 5, 2, float("nan")], -1)):
        with pytest.raises(AtlasError) as e:
            m.generate_beam(*args)
        assert e.value.code == code
    tiny = modelgen.engine_model(modelgen.make_weights(modelgen.tiny_config(), seed=1), max_batch=2)
    with pytest.raises(AtlasError) as e:
        tiny.generate_beam([1, 2], 3, 2)
    assert e.value.code == -4


def test_beam_search_without_memory():
    W, prompt = _weights("olmo", 2), _prompt(2, 9)
    want = _model(W, 4).generate_beam(prompt, 6, 4)
    m = _model(W, 4)
    for skip in range(6):
        check(load().atlas_debug_fail_allocations(skip, 1))
        try:
            m.generate_beam(prompt, 6, 4)
            failed = False
        except AtlasError as e:
            failed = True
            assert e.code == -3
        finally:
            check(load().atlas_debug_fail_allocations(0, 0))
        if not failed:
            break
    assert m.generate_beam(prompt, 6, 4) == want


def test_beam_search_refuses_what_it_has_no_memory_for():
    """A first search allocates a block on the host and four on the device, in turn.  Each fails once, and the search with it:
    the first at once, each other after the one before it; then there is nothing left to allocate."""
    W, prompt = _weights("olmo", 2), _prompt(2, 9)
    want = _model(W, 4).generate_beam(prompt, 6, 4)
    m, codes, got = _model(W, 4), [], None
    for skip in [0] + [1] * 20:
        check(load().atlas_debug_fail_allocations(skip, 1))
        try:
            got = m.generate_beam(prompt, 6, 4)
            break
        except AtlasError as e:
            codes.append(e.code)
        finally:
            check(load().atlas_debug_fail_allocations(0, 0))
    assert len(codes) >= 5 and set(codes) == {-3} and got == want
    assert m.generate_beam(prompt, 6, 4) == want


def test_infer_command_with_beams(tmp_path):
    from atlas_amd import cli
    from tests import ckptgen
    cfg = modelgen.olmo3_small_config(max_seq=256)
    W = modelgen.make_weights(cfg, seed=97)
    conf = ckptgen.olmo3_config_json(cfg)
    conf.update(num_attention_heads=cfg["n_heads"], num_key_value_heads=cfg["n_kv_heads"],
                intermediate_size=cfg["ffn_hidden"], max_position_embeddings=cfg["max_seq"])
    ckptgen.write_dir(str(tmp_path), ckptgen.hf_tensors(W), config=conf)
    lines = []
    rep = cli.run_infer(cli.parse_args(["--weights", str(tmp_path), "--model", "auto", "--prompt", "beam", "--max-tokens", "7",
                                        "--beams", "3"]), out=lines.append)
    m = _model(W, 3)
    want = m.generate_beam(list(b"beam"), 7, 3)
    assert rep["tokens"] == want[0][0]
    assert sum("  Beam  " in x for x in lines) == 3
