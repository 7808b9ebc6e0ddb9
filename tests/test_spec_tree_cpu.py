"""Trees of drafts and sampled drafts on the CPU twin: tokens are those of plain decoding, greedy or sampled with the same seed."""
import torch

from coffin_b200.config import preset
from coffin_b200.engine.config import EngineConfig
from coffin_b200.engine.llm_engine import LLMEngine
from coffin_b200.engine.sequence import SamplingParams
from coffin_b200.oracle import ops as O
from coffin_b200.oracle.engine_model import OracleEngineModel
from coffin_b200.utils.suffix import SuffixDrafter
from coffin_b200.weights.init import random_state_dict

CFG = preset("tiny")
SD = random_state_dict(CFG, 0)


def _engine(num_slots=4, num_blocks=None, **kw):
    model = OracleEngineModel(CFG, SD, max_seq=512, num_slots=num_slots, num_blocks=num_blocks)
    return LLMEngine(model, EngineConfig(max_seq=512, max_num_seqs=num_slots, graph=False, **kw))


def _branching(seed: int, n: int = 60) -> list[int]:
    """A unit that is repeated with one of two endings, so that suffixes have several continuations."""
    g = torch.Generator().manual_seed(seed)
    unit, ends = torch.randint(0, CFG.vocab_size, (4,), generator=g).tolist(), torch.randint(0, CFG.vocab_size, (2, 2), generator=g).tolist()
    out: list[int] = []
    while len(out) < n:
        out += unit + ends[int(torch.randint(0, 2, (1,), generator=g))]
    return out[:n]


def test_drafted_trees_hold_the_chain_and_branch_where_continuations_differ():
    d = SuffixDrafter(max_match=4, min_match=2)
    d.observe([5, 6, 7, 8, 9, 5, 6, 7, 8, 1, 5, 6, 7])
    tokens, parents = d.draft_tree(3, 16)
    assert tokens[:3] == d.draft(3) == [8, 1, 5]
    assert all(-1 <= p < j for j, p in enumerate(parents))
    paths = set()
    for j in range(len(tokens)):
        path, k = [], j
        while k >= 0:
            path.insert(0, tokens[k])
            k = parents[k]
        paths.add(tuple(path))
    assert (8, 1, 5) in paths and (8, 9, 5) in paths
    assert len({(p, t) for p, t in zip(parents, tokens)}) == len(tokens), "siblings differ"
    assert d.draft_tree(3, 2) == (tokens[:2], parents[:2])
    assert d.draft_tree(0, 5) == ([], []) == d.draft_tree(3, 0)
    d.reset()
    assert d.draft_tree(3, 5) == ([], [])


def test_draw_and_walk():
    logits = torch.log(torch.tensor([0.1, 0.2, 0.3, 0.4]))
    assert [O.draw(logits, 1.0, u) for u in (0.0, 0.0999, 0.1001, 0.31, 0.61, 0.999999, 1.0)] == [0, 0, 1, 2, 3, 3, 3]
    assert O.draw(logits, 0.0, 0.1) == 3
    rows = logits.repeat(4, 1)
    assert O.tree_walk(rows, [9, 1, 2, 2], [-1, 0, 0, 2], 1.0, [0.5, 0.5, 0.05]) == ([0, 2, 3], 0)
    assert O.tree_walk(rows, [9, 1, 3, 2], [-1, 0, 0, 2], 0.0, []) == ([0, 2], 3)


@torch.no_grad()
def test_trees_of_drafts_give_the_tokens_of_plain_greedy_decoding():
    prompts = [_branching(1), _branching(2, 45), _branching(3, 70)]
    ref = [s.output for s in _engine().generate(prompts, SamplingParams(max_tokens=24))]
    for kw in ({"spec_tree": 7}, {"spec_tree": 12, "spec_batch": True}):
        eng = _engine(spec_k=4, **kw)
        seqs = [eng.add_request(p, SamplingParams(max_tokens=24)) for p in prompts] if kw.get("spec_batch") else None
        if seqs is None:
            seqs = [eng.generate([p], SamplingParams(max_tokens=24))[0] for p in prompts]
        while any(not s.finished for s in seqs):
            eng.step()
        assert [s.output for s in seqs] == ref
        st = eng.runner.stats()["spec"]
        assert st["steps"] > 0 and st["accepted"] > 0
        eng.bm.pool.check()


@torch.no_grad()
def test_sampled_requests_draft_and_keep_their_tokens():
    """Hot rows beside greedy ones: the tokens of every row are those it gets alone, without drafts."""
    prompts = [_branching(4), _branching(5, 50), _branching(6, 66)]
    params = [SamplingParams(max_tokens=16, temperature=0.02, seed=7), SamplingParams(max_tokens=16), SamplingParams(max_tokens=16, temperature=0.9, seed=9)]
    ref = [_engine().generate([p], q)[0].output for p, q in zip(prompts, params)]
    for kw in ({"spec_sample": True}, {"spec_sample": True, "spec_tree": 10}, {"spec_tree": 10}):
        eng = _engine(spec_k=3, spec_batch=True, **kw)
        seqs = [eng.add_request(p, q) for p, q in zip(prompts, params)]
        while any(not s.finished for s in seqs):
            eng.step()
        assert [s.output for s in seqs] == ref, kw
        assert (seqs[0].spec_drafted > 0) == ("spec_sample" in kw) and seqs[1].spec_drafted > 0
        if "spec_sample" in kw:
            assert seqs[0].spec_accepted > 0, "a cold row follows its repetitive prompt"
        eng.bm.pool.check()


@torch.no_grad()
def test_trees_stop_at_eos_and_the_window_and_survive_a_tight_pool():
    p = _branching(8)
    ref = _engine().generate([p], SamplingParams(max_tokens=30))[0].output
    eos = ref[11]
    s = _engine(spec_k=4, spec_tree=9).generate([p], SamplingParams(max_tokens=30, eos=(eos,)))[0]
    assert s.output == ref[:ref.index(eos)] and s.finish_reason == "stop"
    prompts = [_branching(k, 120) for k in (11, 12, 13)]
    ref = [_engine().generate([q], SamplingParams(max_tokens=14))[0].output for q in prompts]
    eng = _engine(num_slots=3, num_blocks=9, prefix_cache=False, spec_k=3, spec_batch=True, spec_tree=6)
    seqs = [eng.add_request(q, SamplingParams(max_tokens=14)) for q in prompts]
    for _ in range(2000):
        if all(s.finished for s in seqs):
            break
        eng.step()
        eng.bm.pool.check()
    assert [s.output for s in seqs] == ref and eng.bm.pool.used_blocks == 0
    long = _branching(14, 500)
    s = _engine(spec_k=7, spec_tree=20).generate([long], SamplingParams(max_tokens=50))[0]
    assert s.finish_reason == "window" and s.output == _engine().generate([long], SamplingParams(max_tokens=50))[0].output
