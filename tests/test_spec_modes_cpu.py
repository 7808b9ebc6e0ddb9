"""Which way a speculative step goes: trees where the model verifies them, chains where it does not."""
from types import SimpleNamespace

import pytest
import torch

from coffin_b200.config import preset
from coffin_b200.engine.config import EngineConfig
from coffin_b200.engine.llm_engine import LLMEngine
from coffin_b200.engine.sequence import SamplingParams
from coffin_b200.oracle.engine_model import OracleEngineModel
from coffin_b200.weights.init import random_state_dict

CFG = preset("tiny")
SD = random_state_dict(CFG, 0)


class ChainsOnly(OracleEngineModel):
    """What a model over several ranks is: it has the tree pass, but not for its layout."""
    verifies_trees = False

    def verify_tree(self, rows):
        raise NotImplementedError("a verify pass over trees is single-GPU")


def _engine(cls=OracleEngineModel, **kw):
    return LLMEngine(cls(CFG, SD, max_seq=512, num_slots=4), EngineConfig(max_seq=512, max_num_seqs=4, graph=False, **kw))


def _repetitive(seed: int, n: int = 60) -> list[int]:
    g = torch.Generator().manual_seed(seed)
    unit = torch.randint(0, CFG.vocab_size, (6,), generator=g).tolist()
    return (unit * 20)[:n]


@torch.no_grad()
@pytest.mark.parametrize("kw", [{"spec_tree": 7}, {"spec_sample": True}, {"spec_tree": 9, "spec_sample": True}])
def test_a_model_without_tree_passes_drafts_chains(kw):
    """Greedy rows draft chains, sampled ones do not draft, and all finish with the tokens of plain decoding."""
    prompts = [_repetitive(1), _repetitive(2, 50)]
    params = [SamplingParams(max_tokens=16), SamplingParams(max_tokens=16, temperature=0.05, seed=3)]
    ref = [_engine().generate([p], q)[0].output for p, q in zip(prompts, params)]
    eng = _engine(ChainsOnly, spec_k=3, spec_batch=True, **kw)
    assert not eng.runner.tree_capable and not eng.runner.tree_drafts
    seqs = [eng.add_request(p, q) for p, q in zip(prompts, params)]
    assert eng.runner.spec_k_of(seqs[0]) == 3 and eng.runner.spec_k_of(seqs[1]) == 0
    while any(not s.finished for s in seqs):
        eng.step()
    assert [s.output for s in seqs] == ref
    assert seqs[0].spec_accepted > 0 and seqs[1].spec_drafted == 0


def test_the_device_model_verifies_trees_on_one_rank_only():
    from coffin_b200.models.qwen35.model import Qwen35Model
    says = Qwen35Model.verifies_trees.fget
    comm = object()
    assert says(SimpleNamespace(tp=None, tp_world=1, ep_world=1)) and says(SimpleNamespace(tp=comm, tp_world=1, ep_world=1))
    assert not says(SimpleNamespace(tp=comm, tp_world=2, ep_world=1)) and not says(SimpleNamespace(tp=comm, tp_world=1, ep_world=2))


class TwoSamplers(OracleEngineModel):
    """A model whose plain draw differs from the draw of its tree pass."""

    def sample(self, logits, temps, us):
        out = super().sample(logits, temps, us)
        if temps is None:
            return out
        self.plain = getattr(self, "plain", 0) + 1
        return torch.tensor([(int(t) + (temp > 0)) % logits.shape[1] for t, temp in zip(out, temps)])

    def draw(self, logits, temps, us):
        self.drawn = getattr(self, "drawn", 0) + 1
        return super().sample(logits, temps, us)


@torch.no_grad()
def test_a_sampled_request_has_one_sampler_whether_or_not_a_step_drafted():
    """With speculation over trees every token of a request is drawn alike: the first one, those of steps without drafts and those of tree
    steps.  Without it the plain draw is used, as ever."""
    prompts = [_repetitive(4), _repetitive(5, 50)]
    params = [SamplingParams(max_tokens=24, temperature=0.05, seed=3), SamplingParams(max_tokens=24, temperature=0.9, seed=5)]
    ref = [_engine().generate([p], q)[0].output for p, q in zip(prompts, params)]        # the oracle's draws throughout
    for kw in ({"spec_sample": True}, {"spec_tree": 7}, {"spec_tree": 7, "spec_sample": True}):
        eng = _engine(TwoSamplers, spec_k=3, spec_batch=True, **kw)
        seqs = [eng.add_request(p, q) for p, q in zip(prompts, params)]
        while any(not s.finished for s in seqs):
            eng.step()
        assert [s.output for s in seqs] == ref, kw
        assert not hasattr(eng.model, "plain") and eng.model.drawn > 0
    eng = _engine(TwoSamplers, spec_k=3, spec_batch=True)
    eng.generate(prompts[:1], params[0])
    assert eng.model.plain > 0 and not hasattr(eng.model, "drawn")


@torch.no_grad()
def test_without_a_number_of_tree_nodes_a_row_drafts_one_chain():
    """Continuations that end with the history leave room for others, which branch where the tree flag is set and nowhere else."""
    prompt = [5, 6, 7, 8, 9, 5, 6, 7, 8, 1, 2, 5, 6, 7, 8, 1, 5, 6]
    for q in (SamplingParams(max_tokens=4), SamplingParams(max_tokens=4, temperature=0.5, seed=1)):
        drafted = {}
        for n in (0, 12):
            eng = _engine(spec_k=7, spec_sample=True, spec_tree=n)
            seq = eng.add_request(prompt, q)
            (drafted[n],) = eng.runner.draft_trees([seq])
        tokens, parents = drafted[0]
        assert tokens == [7, 8, 1, 5, 6] == seq.drafter.draft(7) and parents == [-1, 0, 1, 2, 3]
        assert drafted[12][0][:5] == tokens and len(drafted[12][0]) > 5


class FewRows(ChainsOnly):
    """Over several ranks a verify pass has at most 8 token rows, of a power of two of sequences."""
    verify_rows = 8
    widest = 0

    def verify_batch(self, rows):
        n = 1
        while n < len(rows):
            n *= 2
        if n * len(rows[0][0]) > 8:
            raise NotImplementedError("a verify pass of more than 8 token rows is single-GPU")
        self.widest = max(self.widest, n * len(rows[0][0]))
        return super().verify_batch(rows)


class Knowing:
    """Drafts a request's own tokens, so that chains are as long as they may be."""

    def __init__(self, prompt, output):
        self.want, self.seen = list(prompt) + list(output), 0

    def observe(self, tokens):
        self.seen += len(tokens)

    def draft(self, k):
        return self.want[self.seen:self.seen + k]


@torch.no_grad()
@pytest.mark.parametrize("n", [1, 2, 3, 4])
@pytest.mark.parametrize("kw", [{}, {"spec_tree": 9}], ids=["chain", "tree"])
def test_chains_of_several_rows_fit_the_verify_pass_of_the_model(n, kw):
    prompts = [_repetitive(20 + i, 48 + i) for i in range(n)]
    ref = [_engine().generate([p], SamplingParams(max_tokens=12))[0].output for p in prompts]
    eng = _engine(FewRows, spec_k=7, spec_batch=True, **kw)
    seqs = [eng.add_request(p, SamplingParams(max_tokens=12)) for p in prompts]
    for s, r in zip(seqs, ref):
        s.drafter, s.drafter_seen = Knowing(s.prompt, r), 0
    while any(not s.finished for s in seqs):
        eng.step()
    assert [s.output for s in seqs] == ref
    assert eng.model.widest == 8 and eng.runner.stats()["spec"]["accepted"] > 0


def test_rows_of_a_verify_pass_on_the_device():
    from coffin_b200.models.qwen35.model import Qwen35Model
    says = Qwen35Model.verify_rows.fget
    comm = object()
    assert says(SimpleNamespace(tp=None, tp_world=1, ep_world=1)) == 64 == says(SimpleNamespace(tp=comm, tp_world=1, ep_world=1))
    assert says(SimpleNamespace(tp=comm, tp_world=2, ep_world=1)) == 8 == says(SimpleNamespace(tp=comm, tp_world=1, ep_world=2))
