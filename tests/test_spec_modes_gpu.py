"""Draws of sampled requests on the device: steps with and without drafts draw alike."""
from types import SimpleNamespace

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale,T", [(3.0, 0.8), (3.0, 1.3), (1.0, 1.0)])
def test_plain_steps_and_tree_steps_draw_the_same_tokens(scale, T):
    """4096 draws among 151936 tokens: one row at a time as a plain step draws them, and along 64 chains of drafts whose tokens are those
    draws, which have to be kept to their ends.  (Sums of the two calls may be cut differently; they are 64-bit, so a draw differs with a
    probability of about 1e-11.)"""
    from coffin_b200.models.qwen35.model import Qwen35Model
    from coffin_b200.ops import tree
    R = C = 64
    V = 151936
    g = torch.Generator(device="cuda").manual_seed(int(10 * scale + 100 * T))
    logits = torch.randn(R, 1, V, generator=g, device="cuda") * scale
    u = torch.rand(R, C, generator=g, device="cuda")
    model = SimpleNamespace(device="cuda")
    draws = torch.stack([Qwen35Model.draw(model, logits[r].expand(C, V), [T] * C, u[r].tolist()) for r in range(R)])
    tokens = torch.zeros(R, C, dtype=torch.int64, device="cuda")
    tokens[:, 1:] = draws[:, :-1]
    anc = torch.tensor([tree.path_words(list(range(-1, C - 1)))] * R, dtype=torch.int64, device="cuda")
    _path, steps, nxt = tree.verify_tree(logits.expand(R, C, V), tokens, anc, torch.full((R,), T, device="cuda"), u)
    assert steps.tolist() == [C] * R
    assert torch.equal(nxt, draws[:, -1])


def test_a_plain_step_draws_hot_and_greedy_rows_together():
    from coffin_b200.models.qwen35.model import Qwen35Model
    g = torch.Generator(device="cuda").manual_seed(2)
    logits = torch.randn(3, 5000, generator=g, device="cuda")
    logits[1, 77] = logits[1, 4000] = 50.0
    model = SimpleNamespace(device="cuda")
    got = Qwen35Model.draw(model, logits, [0.7, 0.0, 1.0], [0.25, 0.9, 0.999])
    for r, (T, u) in enumerate([(0.7, 0.25), (0.0, 0.9), (1.0, 0.999)]):
        if T <= 0:
            want = 77
        else:
            cdf = torch.softmax(logits[r].double() / T, 0).cumsum(0)
            want = int(torch.searchsorted(cdf, torch.tensor(u, dtype=torch.float32, device="cuda").double() * cdf[-1], right=True))
        assert int(got[r]) == want, r


def _rel(a, b):
    return ((a.float() - b.float()).abs().max() / b.float().abs().max()).item()


@torch.no_grad()
@pytest.mark.parametrize("kv_dtype", ["bf16", "int8"])
def test_a_committed_path_with_drafts_that_collide(kv_dtype):
    """The drafts of one path are the model's own tokens, and no other node carries one: the path is taken to its end and committed, where an
    earlier sibling of it had the same token too.  Bounds as for a verify pass against steps."""
    from coffin_b200.config import preset
    from coffin_b200.models.qwen35.model import Qwen35Model
    from coffin_b200.weights.init import random_state_dict
    cfg = preset("tiny")
    spec, step = (Qwen35Model(cfg, random_state_dict(cfg, 0), max_seq=512, num_slots=2, kv_dtype=kv_dtype) for _ in range(2))
    parents = [-1, 0, 0, 0, 1, 4, 5, 3, 7, 8, 6]
    g = torch.Generator().manual_seed(21)
    n, table = 61, list(range(1, 9))                       # the tree lies across a page's end
    prompt = torch.randint(0, cfg.vocab_size, (n,), generator=g)
    bt = torch.tensor(table, dtype=torch.int32, device="cuda")
    for m in (spec, step):
        m.zero_state(0)
        m.prefill(prompt.cuda(), 0, 0, bt, want_logits=False)
    toks = torch.randint(0, cfg.vocab_size, (len(parents),), generator=g).tolist()
    toks[1] = toks[2]                                      # siblings that are equal
    row = [(toks, parents, n, 0, table, 0)]
    want, at = [0], 0
    while True:
        kids = [j for j in range(len(parents)) if parents[j] == at]
        if not kids:
            break
        own = int(spec.verify_tree(row)[0, at].argmax())
        for j in kids[:-1]:                                # the first node with the token is taken: only the last one may carry it
            if toks[j] == own:
                toks[j] = (own + 1) % cfg.vocab_size
        toks[kids[-1]] = own
        at = kids[-1]
        want.append(at)
    assert want == [0, 3, 7, 8, 9]
    logits = spec.verify_tree(row).clone()
    paths, nxt = spec.accept_tree([0.0], [[]])
    assert paths == [want] and nxt == [int(logits[0, want[-1]].argmax())]
    spec.commit_tree()
    for i, j in enumerate(want):
        step.set_rows(1, [toks[j]], [n + i], [0], [table])
        step.decode(1, graph=False)
    for li in range(spec.state.shape[0]):
        assert _rel(spec.state[li, 0], step.state[li, 0]) < 3e-2, li
    outs = []
    for m in (spec, step):
        m.set_rows(1, nxt, [n + len(want)], [0], [table])
        outs.append(m.decode(1, graph=False)[1][0].clone())
    assert _rel(*outs) < 4e-2


@torch.no_grad()
@pytest.mark.parametrize("kv_dtype", ["bf16", "int8"])
@pytest.mark.parametrize("kw", [{"spec_tree": 12}, {"spec_sample": True}, {"spec_tree": 15, "spec_sample": True}], ids=["tree", "sample", "both"])
def test_engine_tokens_are_the_draws_from_the_logits_of_their_steps(kw, kv_dtype):
    """Every tree step: path and token are those of the 64-bit walk on the host over the logits of that pass, for greedy and sampled rows alike;
    drafts are accepted.  Every greedy token is, to the roundings of two pipelines, the arg-max of plain decoding over pages of the same type."""
    from coffin_b200.config import preset
    from coffin_b200.engine.config import EngineConfig
    from coffin_b200.engine.llm_engine import LLMEngine
    from coffin_b200.engine.sequence import SamplingParams
    from coffin_b200.models.qwen35.model import Qwen35Model
    from coffin_b200.oracle import ops as O
    from coffin_b200.weights.init import random_state_dict
    cfg = preset("tiny")
    sd = random_state_dict(cfg, 0)
    model, step = (Qwen35Model(cfg, sd, max_seq=512, num_slots=4, kv_dtype=kv_dtype) for _ in range(2))
    eng = LLMEngine(model, EngineConfig(max_seq=512, max_num_seqs=4, spec_k=3, spec_batch=True, **kw))
    seen = []
    verify, accept = model.verify_tree, model.accept_tree
    passes = []

    def spy_verify(rows):
        lg = verify(rows)
        passes.append((rows, lg.clone()))
        return lg

    def spy_accept(temps, us):
        got = accept(temps, us)
        seen.append((*passes[-1], temps, us, got))
        return got

    model.verify_tree, model.accept_tree = spy_verify, spy_accept
    g = torch.Generator().manual_seed(6)
    prompts = []
    for i in range(4):
        unit = torch.randint(0, cfg.vocab_size, (5 + i,), generator=g).tolist()
        prompts.append((unit * 12)[:48 + 3 * i])
    params = [SamplingParams(max_tokens=20), SamplingParams(max_tokens=20, temperature=0.02, seed=1), SamplingParams(max_tokens=20),
              SamplingParams(max_tokens=20, temperature=0.8, seed=2)]
    seqs = [eng.add_request(p, q) for p, q in zip(prompts, params)]
    while any(not s.finished for s in seqs):
        eng.step()
    assert seen and eng.runner.stats()["spec"]["accepted"] > 0
    for rows, lg, temps, us, (paths, last) in seen:
        for i, row in enumerate(rows):
            host = [float(torch.tensor(u, dtype=torch.float32)) for u in us[i]]
            assert O.tree_walk(lg[i].cpu(), row[0], row[1], temps[i], host) == (paths[i], last[i])
    table = list(range(1, 9))
    bt = torch.tensor(table, dtype=torch.int32, device="cuda")
    for s in (seqs[0], seqs[2]):
        p = s.prompt
        step.zero_state(0)
        lg = step.prefill(torch.tensor(p).cuda(), 0, 0, bt)
        for i, tok in enumerate(s.output):
            lg = lg.reshape(-1)
            assert float(lg.max() - lg[tok]) <= 2 * 4e-2 * float(lg.abs().max()), i
            step.set_rows(1, [tok], [len(p) + i], [0], [table])
            lg = step.decode(1, graph=False)[1][0].clone()
