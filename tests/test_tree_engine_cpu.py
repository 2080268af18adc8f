"""Speculative decoding over trees of drafts in the generation engine (CPU path): the output is the target's own, whatever
the drafts are, and both caches stay consistent."""
import pytest
import torch

from antfly_b200.models.llama import LlamaConfig, LlamaModel
from antfly_b200.runtime.engine import LLMEngine
from antfly_b200.runtime.kv_cache import KvOutOfBlocks
from antfly_b200.runtime.sampling_params import SamplingParams

PROMPTS = [[7, 8, 9, 10] * 5, [100, 101, 102], [42] * 33]


def _model(seed=0, **kw):
    return LlamaModel.random_init(LlamaConfig.tiny(num_hidden_layers=2, **kw), device="cpu", seed=seed)


def _engine(num_blocks=64, **kw):
    return LLMEngine(_model(), num_blocks=num_blocks, page=16, max_batch=4, max_step_tokens=64, use_cuda_graph=False, **kw)


@pytest.fixture(scope="module")
def plain():
    return [r.token_ids for r in _engine().generate(PROMPTS, SamplingParams(max_tokens=14))]


@pytest.mark.parametrize("tree", [(2,), (3, 2, 1), (1, 1, 1, 1)])
def test_trees_from_the_first_layers_reproduce_greedy_output(plain, tree):
    eng = _engine(draft_layers=1, spec_tree=tree)
    assert [r.token_ids for r in eng.generate(PROMPTS, SamplingParams(max_tokens=14))] == plain
    st = eng.spec
    assert st.rounds > 0 and st.drafted == st.matched + st.rejected and st.accepted <= st.matched + st.corrections + st.bonus
    assert eng.cache.alloc.free_blocks == 64


def test_trees_from_a_separate_model_reproduce_greedy_output_and_leave_both_pools_empty(plain):
    eng = _engine(draft_model=_model(seed=5), spec_tree=(4, 2))
    assert [r.token_ids for r in eng.generate(PROMPTS, SamplingParams(max_tokens=14))] == plain
    assert eng.cache.alloc.free_blocks == 64 and eng.draft_cache.alloc.free_blocks == 64


def test_a_draft_that_equals_the_target_is_accepted_to_the_last_level(plain):
    """Every round accepts a full path, so each next one depends on the rows that were moved and on the draft cache's
    catch-up of the last level."""
    eng = _engine(draft_model=_model(), spec_tree=(2, 2, 1))
    assert [r.token_ids for r in eng.generate(PROMPTS, SamplingParams(max_tokens=14))] == plain
    assert eng.spec.bonus > 0 and eng.spec.corrections == 0


def test_a_tree_of_one_branch_per_level_drafts_what_a_chain_drafts(plain):
    chain, tree = _engine(draft_layers=1, spec_k=3), _engine(draft_layers=1, spec_tree=(1, 1, 1))
    sp = SamplingParams(max_tokens=14)
    assert [r.token_ids for r in chain.generate(PROMPTS, sp)] == [r.token_ids for r in tree.generate(PROMPTS, sp)] == plain
    assert (chain.spec.drafted, chain.spec.matched) == (tree.spec.drafted, tree.spec.matched)


@pytest.mark.parametrize("kv_dtype", ["fp8", "int8"])
def test_trees_over_a_quantised_cache(kv_dtype):
    sp = SamplingParams(max_tokens=8)
    plain = [r.token_ids for r in _engine(kv_dtype=kv_dtype).generate(PROMPTS[:2], sp)]
    eng = _engine(kv_dtype=kv_dtype, draft_layers=1, spec_tree=(2, 1))
    assert [r.token_ids for r in eng.generate(PROMPTS[:2], sp)] == plain


def test_a_sliding_window_counts_positions_along_the_path():
    prompts, sp = [[3, 4, 5, 6] * 6], SamplingParams(max_tokens=10)
    make = lambda **kw: LLMEngine(_model(sliding_window=12), num_blocks=32, page=16, max_batch=2, max_step_tokens=64,
                                  use_cuda_graph=False, **kw)
    plain = [r.token_ids for r in make().generate(prompts, sp)]
    assert [r.token_ids for r in make(draft_layers=1, spec_tree=(3, 2)).generate(prompts, sp)] == plain


def test_stops_and_limits_inside_an_accepted_path(plain):
    eng = _engine(draft_model=_model(), spec_tree=(2, 1, 1))
    res = eng.generate([PROMPTS[0]], SamplingParams(max_tokens=14, stop_token_ids=[plain[0][2]]))[0]
    assert res.token_ids == plain[0][:plain[0].index(plain[0][2]) + 1] and res.finish_reason == "stop"
    assert [len(r.token_ids) for r in eng.generate(PROMPTS[:2], SamplingParams(max_tokens=2))] == [2, 2]
    assert eng.cache.alloc.free_blocks == 64


def test_a_tree_that_does_not_fit_behind_a_sequence_gives_way_to_a_chain(plain):
    eng = LLMEngine(_model(), num_blocks=16, page=16, max_batch=4, max_step_tokens=64, use_cuda_graph=False, max_seq_len=48,
                    draft_layers=1, spec_k=1, spec_tree=(4, 2, 2))
    assert eng.generate([PROMPTS[0]], SamplingParams(max_tokens=14))[0].token_ids == plain[0]


def test_an_exhausted_pool_leaves_the_sequences_as_they_were():
    eng = _engine(num_blocks=4, draft_layers=1, spec_tree=(8, 4))
    rid = eng.add_request([5] * 40, SamplingParams(max_tokens=30))
    with pytest.raises(KvOutOfBlocks):
        while eng.has_work():
            eng.step()
    r = eng.reqs[rid]
    assert eng.cache.alloc.length(rid) == len(r.prompt) + len(r.out) - 1


DRAFTS = [lambda: dict(draft_layers=1), lambda: dict(draft_model=_model()), lambda: dict(draft_model=_model(), draft_num_blocks=3)]


@pytest.mark.parametrize("draft", DRAFTS)
@pytest.mark.parametrize("form", [dict(spec_tree=(8, 2)), dict(spec_tree=(2, 1)), dict(spec_k=4)])
def test_a_pool_that_holds_the_continuation_but_not_the_drafts(draft, form):
    """Four blocks hold the 63 tokens of a request to the last; rounds whose drafts do not fit them, or a separate draft's
    pool, give way to chains and in the end to plain steps."""
    sp, prompt = SamplingParams(max_tokens=24), [PROMPTS[0] * 2]
    plain = [r.token_ids for r in _engine(num_blocks=4).generate(prompt, sp)]
    eng = _engine(num_blocks=4, **{**draft(), **form})
    assert [r.token_ids for r in eng.generate(prompt, sp)] == plain and len(plain[0]) == 24
    assert eng.cache.alloc.free_blocks == 4
    assert eng.draft_cache is None or eng.draft_cache.alloc.free_blocks == eng.draft_cache.num_blocks


@pytest.mark.parametrize("form", [dict(spec_tree=(4, 2)), dict(spec_k=4)])
def test_cached_prefixes_give_way_to_drafts(form):
    """The first prompts' blocks stay cached until the pool is full; the last request still speculates."""
    sp, prompts = SamplingParams(max_tokens=12), [[i + 1] * 32 for i in range(3)] + [PROMPTS[0]]
    plain = [_engine(num_blocks=8).generate([p], sp)[0].token_ids for p in prompts]
    eng = _engine(num_blocks=8, draft_layers=1, prefix_cache=True, **form)
    got = []
    for p in prompts:
        before = eng.spec.rounds
        got.append(eng.generate([p], sp)[0].token_ids)
        assert eng.spec.rounds > before
    assert got == plain and eng.prefix.evictions > 0


def test_a_chain_at_the_end_of_the_block_table_gives_way_to_plain_steps(plain):
    eng = LLMEngine(_model(), num_blocks=16, page=16, max_batch=4, max_step_tokens=64, use_cuda_graph=False, max_seq_len=48,
                    draft_layers=1, spec_k=4)
    want = LLMEngine(_model(), num_blocks=16, page=16, max_batch=4, max_step_tokens=64, use_cuda_graph=False, max_seq_len=48)
    sp = SamplingParams(max_tokens=28)
    assert eng.generate([PROMPTS[0]], sp)[0].token_ids == want.generate([PROMPTS[0]], sp)[0].token_ids


def test_sampled_requests_run_over_trees():
    sp = SamplingParams(max_tokens=6, temperature=0.8, top_k=20, repetition_penalty=1.1, seed=3)
    out = _engine(draft_layers=1, spec_tree=(2, 2)).generate(PROMPTS[:2], sp)
    assert all(len(r.token_ids) == 6 and all(0 <= t < 512 for t in r.token_ids) for r in out)


@pytest.mark.parametrize("penalty", [dict(repetition_penalty=1.2), dict(frequency_penalty=0.5), dict(presence_penalty=0.7)])
@pytest.mark.parametrize("tree", [(2, 2, 2), (3, 1, 1, 1)])
def test_penalties_count_the_drafts_in_front_of_a_node(penalty, tree):
    """A twin of the target drafts long accepted paths; the token behind each of their nodes is penalised for the drafts on
    the way, so that the output is that of the engine without a draft."""
    sp = SamplingParams(max_tokens=14, **penalty)
    plain = [r.token_ids for r in _engine().generate(PROMPTS, sp)]
    for kw in (dict(draft_model=_model()), dict(draft_layers=1)):
        eng = _engine(spec_tree=tree, **kw)
        assert [r.token_ids for r in eng.generate(PROMPTS, sp)] == plain
    mixed = [sp, SamplingParams(max_tokens=14), sp]               # requests of both kinds in a round
    plain = [r.token_ids for r in _engine().generate(PROMPTS, mixed)]
    assert [r.token_ids for r in _engine(spec_tree=tree, draft_model=_model()).generate(PROMPTS, mixed)] == plain


@pytest.mark.parametrize("penalty", [dict(repetition_penalty=1.2), dict(frequency_penalty=0.5)])
def test_penalties_count_the_drafts_in_front_of_a_chains_row(penalty):
    sp = SamplingParams(max_tokens=14, **penalty)
    plain = [r.token_ids for r in _engine().generate(PROMPTS, sp)]
    for kw in (dict(draft_model=_model()), dict(draft_layers=1)):
        assert [r.token_ids for r in _engine(spec_k=3, **kw).generate(PROMPTS, sp)] == plain


def test_refusals():
    with pytest.raises(ValueError, match="needs a draft"):
        _engine(spec_tree=(2,))
    with pytest.raises(ValueError, match="at least one branch"):
        _engine(draft_layers=1, spec_tree=(2, 0))
    with pytest.raises(ValueError, match="at most 256 nodes"):
        _engine(draft_layers=1, spec_tree=(16, 16))
    sinks = LlamaModel.random_init(LlamaConfig.tiny(num_hidden_layers=2, attn_logit_softcapping=30.0), device="cpu", seed=0)
    with pytest.raises(ValueError, match="not available"):
        LLMEngine(sinks, num_blocks=8, page=16, max_batch=2, max_step_tokens=64, use_cuda_graph=False, draft_layers=1,
                  spec_tree=(2,))
    eng = _engine(draft_layers=1, spec_tree=(2,))
    eng.set_spec_tree(())
    assert eng.spec_tree == ()


def test_more_branches_than_tokens_are_refused():
    few = LlamaModel.random_init(LlamaConfig.tiny(num_hidden_layers=2, vocab_size=64), device="cpu", seed=0)
    make = lambda **kw: LLMEngine(few, num_blocks=16, page=16, max_batch=2, max_step_tokens=64, use_cuda_graph=False,
                                  draft_layers=1, **kw)
    with pytest.raises(ValueError, match="64 branches"):
        make(spec_tree=(2, 65))
    sp = SamplingParams(max_tokens=5)
    assert make(spec_tree=(64, 1)).generate([[7, 8, 9]], sp)[0].token_ids == make().generate([[7, 8, 9]], sp)[0].token_ids
