"""A whole model in 8 bits: beside the same model in its own type, and with a budget."""
import numpy as np
import pytest
import torch

import tiny_configs

pytestmark = pytest.mark.gpu


def _model(name, dtype="bfloat16"):
    from supersonic_b200.config import config_from_dict
    from supersonic_b200.engine import Model
    from supersonic_b200.weights import RandomWeightStore
    cfg, seed, std = tiny_configs.CONFIGS[name]
    c = config_from_dict(cfg)
    return Model.from_config(c, RandomWeightStore(c, seed, device="cuda:0", std=std, norm_jitter=0.0), dtype=dtype, device="cuda:0",
                             max_tokens=2048, max_seq_tokens=512)


def _logits(step, open_, close, sequence, cut):
    """Logits of every token of a sequence that comes as a prompt of ``cut`` tokens and then token by token."""
    from supersonic_b200.engine import StepEntry
    slot = open_()
    rows = [step([StepEntry(slot, sequence[:cut], list(range(cut)))])]
    rows += [step([StepEntry(slot, [t], [0])]) for t in sequence[cut:]]
    close(slot)
    return torch.cat(rows).float().cpu().numpy()


@pytest.mark.parametrize("name,dtype", [("A", "bfloat16"), ("B", "float32"), ("D", "bfloat16"), ("D", "float32"), ("E", "bfloat16")])
def test_logits_beside_the_model_in_its_own_type(name, dtype):
    """8 bits everywhere move the logits by a few per cent of their spread; a misplaced key, scale or channel moves them by all of it."""
    from supersonic_b200.engine.int8_session import Int8Session
    model = _model(name, dtype)
    session = Int8Session(model, max_tokens=1024)
    rng = np.random.default_rng(3)
    sequence = rng.integers(0, model.vocab_size, 150).tolist()
    want = _logits(model.step, model.open_sequence, model.close_sequence, sequence, 130)
    got = _logits(session.step, session.open, session.close, sequence, 130)
    assert np.linalg.norm(got - want) <= 0.15 * np.linalg.norm(want - want.mean(-1, keepdims=True))
    assert sorted(session.free) == list(range(16))
    model.check_errors()


def test_a_batch_generates_what_its_sequences_generate_alone():
    from supersonic_b200.engine.int8_session import Int8Session
    model = _model("D", "float32")
    session = Int8Session(model, max_tokens=1024)
    rng = np.random.default_rng(4)
    prompts = [rng.integers(0, model.vocab_size, n).tolist() for n in (3, 70, 129)]
    together = session.generate(prompts, max_new_tokens=5)
    assert together == [session.generate([p], max_new_tokens=5)[0] for p in prompts]


def test_a_budget_that_is_not_reached_changes_nothing():
    from supersonic_b200.engine.int8_session import Int8Session
    model = _model("E")
    rng = np.random.default_rng(5)
    prompts = [rng.integers(0, model.vocab_size, n).tolist() for n in (100, 40)]
    assert Int8Session(model, 1024).generate(prompts, 6) == Int8Session(model, 1024, budget=200).generate(prompts, 6)


def test_sequences_beyond_their_budget_are_cut_and_go_on(monkeypatch):
    """Held tokens stay within the budget and its slack, positions go on, pages come back; in every layer and head what a cut leaves
    are the values of the tokens it says it kept, to half a code, with the first and the latest among them."""
    from supersonic_b200.csrc import int8_ops
    from supersonic_b200.engine import StepEntry
    from supersonic_b200.engine.int8_session import Int8Session
    model = _model("D", "float32")
    rng = np.random.default_rng(6)
    sequence = rng.integers(0, model.vocab_size, 330).tolist()
    budget, first, recent, cuts = 96, 4, 16, []
    evict = int8_ops.evict

    def read(pages, table, slots, lengths, most):
        out = [torch.zeros((len(slots), most, pages.k.shape[1], pages.k.shape[3]), device="cuda:0") for _ in range(2)]
        int8_ops.read(pages, table, slots, lengths, *out)
        return out

    def watched(pages, table, slots, lengths, new_table, keep, f, r, kept):
        n = int(lengths[0])
        before = read(pages, table, slots, lengths, n)
        evict(pages, table, slots, lengths, new_table, keep, f, r, kept)
        row = torch.zeros(1, dtype=torch.int32, device="cuda:0")
        after = read(pages, new_table, row, row + keep, keep)
        place = kept[0].long()                                   # [kv heads, keep]
        assert (place[:, 1:] > place[:, :-1]).all() and (place[:, :first] == torch.arange(first, device="cuda:0")).all()
        assert (place[:, keep - recent:] == torch.arange(n - recent, n, device="cuda:0")).all()
        for old, new, scale in ((before[0], after[0], pages.k_scale), (before[1], after[1], pages.v_scale)):
            step = scale[new_table[0].long()].transpose(0, 1).reshape(scale.shape[1], -1).repeat_interleave(pages.block, dim=1)[:, :keep]
            want = torch.stack([old[0, place[h], h] for h in range(place.shape[0])])
            assert ((new[0].transpose(0, 1) - want).abs() <= 0.5001 * step[..., None]).all()
        cuts.append(n)
    monkeypatch.setattr(int8_ops, "evict", watched)

    def run():
        session = Int8Session(model, max_tokens=2048, slack=16, budget=budget, first=first, recent=recent)
        slot, rows = session.open(), []
        rows.append(session.step([StepEntry(slot, sequence[:200], [199])]))
        for t in sequence[200:]:
            assert session.length[slot] < budget + 16
            rows.append(session.step([StepEntry(slot, [t], [0])]))
        assert session.position[slot] == 330 and len(session.held[slot]) * 64 >= session.length[slot]
        session.close(slot)
        assert sorted(session.free) == list(range(32))
        return torch.cat(rows)
    logits = run()
    assert cuts == [200] * 2 + [budget + 16] * 2 * (130 // 16) and torch.isfinite(logits).all()
    assert torch.equal(logits, run())


def test_refusals():
    from supersonic_b200.cache import CacheFull
    from supersonic_b200.engine import StepEntry
    from supersonic_b200.engine.int8_session import Int8Session
    import tiny_ronelorn
    from supersonic_b200.engine import Model
    model = _model("A")
    with pytest.raises(ValueError):
        Int8Session(model, 256, budget=10, first=6, recent=6)
    session = Int8Session(model, 128, max_sequences=1)
    with pytest.raises(ValueError):
        session.step([StepEntry(0, [1], [0])])                   # nothing is open
    slot = session.open()
    with pytest.raises(CacheFull):
        session.open()
    with pytest.raises(CacheFull):
        session.step([StepEntry(slot, [1] * 129, [0])])
    cfg, store, _ = tiny_ronelorn.build("A")
    with pytest.raises(ValueError):
        Int8Session(Model.from_config(cfg, store, dtype="bfloat16", device="cuda:0", max_tokens=256, max_seq_tokens=128), 256)


def test_a_refused_step_leaves_the_other_sequences_and_the_session_as_they_were():
    from supersonic_b200.cache import CacheFull
    from supersonic_b200.engine import StepEntry
    from supersonic_b200.engine.int8_session import Int8Session
    model = _model("D", "float32")
    rng = np.random.default_rng(8)
    first, second = (rng.integers(0, model.vocab_size, n).tolist() for n in (60, 70))
    logits = []
    for refused in (False, True):
        session = Int8Session(model, 64 * 5)
        a, b, c = (session.open() for _ in range(3))
        rows = [session.step([StepEntry(a, first, [59])])]
        if refused:
            with pytest.raises(CacheFull):
                session.step([StepEntry(b, second, [69]), StepEntry(c, second * 3, [0])])
            session.close(c)
            with pytest.raises(ValueError):
                session.step([StepEntry(b, second, [69]), StepEntry(c, [1], [0])])
        rows.append(session.step([StepEntry(b, second, [69])]))
        rows += [session.step([StepEntry(a, [5], [0]), StepEntry(b, [6], [0])]) for _ in range(3)]
        logits.append(torch.cat(rows))
    assert torch.equal(*logits)


@pytest.mark.parametrize("step_tokens,most", [(100, 100), (4096, 64 * 8 - 64 * 2 - 129 + 1)])
def test_a_prompt_beyond_the_table_is_cut_on_its_way(monkeypatch, step_tokens, most):
    """A prompt longer than a budget's table, in steps of the model's tokens, or than leaves room for its cut, in steps that do; the same twice."""
    from supersonic_b200.engine import StepEntry
    from supersonic_b200.engine.int8_session import Int8Session
    model = _model("D", "float32")
    monkeypatch.setattr(model, "step_token_budget", step_tokens)
    monkeypatch.setattr(model, "position_limit", None)
    tokens, logits = np.random.default_rng(9).integers(0, model.vocab_size, 500).tolist(), []
    for _ in range(2):
        session, sizes = Int8Session(model, 64 * 8, budget=96, first=4, recent=16, slack=33), []
        run = session._run
        monkeypatch.setattr(session, "_run", lambda packed, cuts: (sizes.append(packed.n_tokens), run(packed, cuts))[1])
        slot = session.open()
        rows = [session.step([StepEntry(slot, tokens, [499, 3, 250])])]
        rows += [session.step([StepEntry(slot, [t], [0])]) for t in (1, 2, 3)]
        assert session.position[slot] == 503 and session.length[slot] < 129 and max(sizes) <= most and sum(sizes) == 503
        session.close(slot)
        assert sorted(session.free) == list(range(8))
        logits.append(torch.cat(rows))
    assert torch.isfinite(logits[0]).all() and logits[0].shape[0] == 6 and torch.equal(*logits)
