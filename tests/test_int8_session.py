"""What an 8-bit session keeps account of (slots, pages, the page table, cuts), on the CPU: its step is replaced by one that writes
every token to its place through the page table and whose logits depend on all that the sequence then holds."""
from types import SimpleNamespace

import pytest
import torch

from supersonic_b200.cache import CacheFull
from supersonic_b200.csrc import int8_ops, ops
from supersonic_b200.engine import StepEntry
from supersonic_b200.engine.int8_session import Int8Session

VOCAB = 97


class Session(Int8Session):
    """Logits of a row: one for (sum over the tokens held up to it of (place + 1) times token) % VOCAB."""

    def __init__(self, max_tokens, step_token_budget=4096, **kw):
        model = SimpleNamespace(device=torch.device("cpu"), dtype=torch.float32, blocks=[], spec=SimpleNamespace(schedule=[]),
                                vocab_size=VOCAB, step_token_budget=step_token_budget, use_graphs=False, _check_positions=lambda n: None)
        super().__init__(model, max_tokens, **kw)
        n_pages = len(self.free)
        self.store = torch.full((n_pages, 64), -1)
        self.layers = [SimpleNamespace(pages=SimpleNamespace(k=torch.zeros((n_pages, 1, 1, 1))))]      # what is cut: the store
        self.steps = []

    def _forward(self, packed, ints):
        rows, flat = [], packed.flat
        T = packed.n_tokens
        place = ints[flat.shape[0]:flat.shape[0] + T].tolist()
        self.steps.append(T)
        for t in range(T):
            slot = int(flat[2 * T + t])
            self.store[self.table[slot, place[t] // 64], place[t] % 64] = int(flat[t])
            held = self.tokens(slot, place[t] + 1)
            assert all(x >= 0 for x in held)
            rows.append(torch.nn.functional.one_hot(torch.tensor(expected(held)), VOCAB).float())
        want = flat[-packed.n_want:] if packed.n_want else []
        return torch.stack([rows[int(w)] for w in want]) if packed.n_want else torch.zeros((0, VOCAB))

    def tokens(self, slot, n):
        """The first ``n`` tokens of a sequence, by the table that a step reads"""
        return [int(self.store[self.table[slot, j // 64], j % 64]) for j in range(n)]

    def account(self):
        return [list(h) for h in self.held], sorted(self.free), self.table.clone(), list(self.position), list(self.length), set(self.open_slots)

    def unchanged_since(self, before):
        now = self.account()
        return all(torch.equal(a, b) if torch.is_tensor(a) else a == b for a, b in zip(before, now)) and torch.equal(self.table, self.table_host)


def expected(tokens):
    return sum((i + 1) * t for i, t in enumerate(tokens)) % VOCAB


@pytest.fixture(autouse=True)
def on_the_host(monkeypatch):
    monkeypatch.setattr(ops, "check_device_errors", lambda device=None: None)


def prompt(n, seed=0):
    return [(7 * seed + 3 * i + i * i) % VOCAB for i in range(n)]


def run(session, *entries):
    """Steps the entries (slot, tokens) and checks every logit."""
    held = {slot: session.tokens(slot, session.length[slot]) for slot, _ in entries}
    logits = session.step([StepEntry(slot, tokens, list(range(len(tokens)))) for slot, tokens in entries])
    want = [expected(held[slot] + list(tokens[:i + 1])) for slot, tokens in entries for i in range(len(tokens))]
    assert logits.argmax(-1).tolist() == want


# ---- steps that are refused ---------------------------------------------------------------------------------------
def test_a_step_refused_for_want_of_pages_changes_nothing():
    session = Session(64 * 4)
    a, b, c = session.open(), session.open(), session.open()
    run(session, (a, prompt(60, 1)))
    before = session.account()
    with pytest.raises(CacheFull):
        session.step([StepEntry(b, prompt(10, 2), [9]), StepEntry(c, prompt(200, 3), [199])])
    assert session.unchanged_since(before)
    run(session, (b, prompt(10, 2)))                               # as if nothing had been: a's page is its own
    run(session, (a, [5]), (b, [6]))
    assert session.tokens(a, 61) == prompt(60, 1) + [5]
    for s in (a, b, c):
        session.close(s)
    assert sorted(session.free) == list(range(4))


def test_a_step_with_a_sequence_that_is_not_open_changes_nothing():
    session = Session(64 * 4, max_sequences=3)
    a, b = session.open(), session.open()
    run(session, (a, prompt(60, 1)))
    before = session.account()
    for other in (2, 3, -1):                                       # not open, and no slot at all
        with pytest.raises(ValueError):
            session.step([StepEntry(b, prompt(10, 2), [9]), StepEntry(other, [1], [0])])
        assert session.unchanged_since(before)
    run(session, (b, prompt(10, 2)), (a, [4]))


def test_a_step_of_tokens_outside_the_vocabulary_changes_nothing():
    session = Session(64 * 4)
    a = session.open()
    before = session.account()
    for bad in ([StepEntry(a, [1, VOCAB], [0])], [StepEntry(a, [], [])], [StepEntry(a, [1], [1])], [StepEntry(a, [1], [0])] * 2, []):
        with pytest.raises(ValueError):
            session.step(bad)
        assert session.unchanged_since(before)
    run(session, (a, [3]))


def test_a_sequence_wider_than_its_table_is_refused_every_time():
    session = Session(64 * 16)
    session.table_host = session.table_host[:, :3].contiguous()     # room for 192 tokens a sequence
    session.table = session.table_host.clone()
    a, b = session.open(), session.open()
    run(session, (a, prompt(64, 1)))
    before = session.account()
    for _ in range(2):
        with pytest.raises(CacheFull):
            session.step([StepEntry(b, prompt(193, 2), [0])])
        assert session.unchanged_since(before)
    run(session, (b, prompt(192, 2)))
    with pytest.raises(CacheFull):
        session.step([StepEntry(b, [1], [0])])
    run(session, (a, [1]))


# ---- generation ---------------------------------------------------------------------------------------------------
def greedy(tokens, n):
    out = []
    for _ in range(n):
        out.append(expected(list(tokens) + out))
    return out


def test_a_refused_generate_gives_its_slots_back():
    session = Session(64 * 8, max_sequences=2)
    prompts = [prompt(5, i) for i in range(3)]
    for refused in (prompts, [[1], []], [prompt(513)]):              # more than there are slots; an empty prompt; no room
        with pytest.raises((CacheFull, ValueError)):
            session.generate(refused, 2)
        assert not session.open_slots and sorted(session.free) == list(range(8))
    assert session.generate(prompts[:2], 4) == [greedy(p, 4) for p in prompts[:2]]


# ---- a budget -----------------------------------------------------------------------------------------------------
@pytest.fixture
def cuts(monkeypatch):
    """Cuts that keep the first ``first`` and the latest tokens, moved as the operator moves them; (tokens before, kept) of each."""
    log = []

    def evict(pages, table, seq_slot, lengths, new_table, keep, first, recent, kept):
        for b, (slot, n) in enumerate(zip(seq_slot.tolist(), lengths.tolist())):
            held = session.tokens(slot, n)
            stay = held if n <= keep else held[:first] + held[n - (keep - first):]
            for j, t in enumerate(stay):
                session.store[new_table[b, j // 64], j % 64] = t
            log.append((n, len(stay)))
    monkeypatch.setattr(int8_ops, "evict", evict)

    def make(*a, **kw):
        nonlocal session
        session = Session(*a, **kw)
        return session
    session = None
    return SimpleNamespace(make=make, log=log)


def test_a_sequence_is_cut_whenever_it_outgrows_its_budget(cuts):
    session = cuts.make(64 * 8, budget=100, slack=20, first=3)
    a = session.open()
    run(session, (a, prompt(150, 1)))
    assert cuts.log == [(150, 100)] and session.length[a] == 100 and session.position[a] == 150
    assert session.tokens(a, 100) == prompt(150, 1)[:3] + prompt(150, 1)[-97:]
    for t in range(45):
        run(session, (a, [t]))
    assert cuts.log == [(150, 100), (120, 100), (120, 100)] and session.position[a] == 195
    session.close(a)
    assert sorted(session.free) == list(range(8))


def test_a_step_whose_cut_has_no_room_changes_nothing(cuts):
    session = cuts.make(192, budget=128, slack=64)                   # three pages, and two more for the cut at 192 tokens
    a = session.open()
    run(session, (a, prompt(191, 1)))
    before = session.account()
    for _ in range(2):
        with pytest.raises(CacheFull):
            session.step([StepEntry(a, [1], [0])])
        assert session.unchanged_since(before) and not cuts.log
    assert session.tokens(a, 191) == prompt(191, 1)


def test_cuts_make_room_for_one_another(cuts):
    """Two sequences of three pages, and room for the pages of one cut: the first one's old pages are the second one's new ones."""
    session = cuts.make(64 * 8, budget=128, slack=1)
    a, b = session.open(), session.open()
    run(session, (a, prompt(128, 1)), (b, prompt(128, 2)))
    run(session, (a, [5]), (b, [6]))
    assert cuts.log == [(129, 128), (129, 128)]
    assert session.tokens(a, 128)[-1] == 5 and session.tokens(b, 128)[-1] == 6 and len(session.free) == 4
    before = session.account()
    c = session.open()
    run(session, (c, prompt(128, 3)))
    with pytest.raises(CacheFull):                                   # two pages for the new tokens, none for a cut
        session.step([StepEntry(a, [7], [0]), StepEntry(b, [8], [0])])
    session.close(c)
    run(session, (a, [7]))
    assert sorted(session.free + session.held[a] + session.held[b]) == list(range(8)) and before[3][a] + 1 == session.position[a]


def test_prompts_longer_than_the_table_are_cut_on_their_way(cuts):
    """A budget bounds what a prompt holds, not how long it is: what does not fit the table runs in chunks with a cut behind each."""
    session = cuts.make(64 * 16, step_token_budget=150, budget=100, slack=30, first=3)
    a, b = session.open(), session.open()
    tokens, other = prompt(1000, 1), prompt(40, 2)
    logits = session.step([StepEntry(b, other, [39]), StepEntry(a, tokens, [999, 0, 500])])
    assert session.position[a] == 1000 and session.position[b] == 40 and all(n <= 150 for n in session.steps)
    assert 100 <= session.length[a] < 130 and session.tokens(a, 3) == tokens[:3]
    assert session.tokens(a, session.length[a])[3:] == tokens[1000 - session.length[a] + 3:]
    assert logits.shape == (4, VOCAB) and logits.argmax(-1).tolist()[0] == expected(other) and logits.argmax(-1).tolist()[2] == expected(tokens[:1])
    assert session.generate([prompt(700, 3)], 3) and not session.open_slots - {a, b}
    session.close(a)
    session.close(b)
    assert sorted(session.free) == list(range(16))


def test_prompts_longer_than_the_cache_are_cut_on_their_way(cuts):
    """Chunks are as small as leaves room for a cut, whatever a step may have."""
    session = cuts.make(64 * 8, step_token_budget=4096, budget=100, slack=30)
    a = session.open()
    session.step([StepEntry(a, prompt(2000, 1), [1999])])
    assert session.position[a] == 2000 and session.length[a] < 130
    assert max(session.steps) <= 64 * 6 - 129 and len(cuts.log) >= 2000 // 384


def test_a_prompt_that_fits_its_table_is_cut_behind_its_last_token(cuts):
    session = cuts.make(64 * 16, step_token_budget=150, budget=100, slack=30)       # a table of 5 pages
    a, b = session.open(), session.open()
    run(session, (a, prompt(320, 1)), (b, prompt(60, 2)))
    assert session.steps == [150, 150, 80] and cuts.log == [(320, 100)]


def test_steps_of_more_tokens_than_the_models_run_in_chunks():
    session = Session(64 * 16, step_token_budget=100)
    a, b = session.open(), session.open()
    run(session, (a, prompt(130, 1)), (b, prompt(250, 2)))
    assert session.steps == [100, 100, 100, 80]
    run(session, *[(s, [1]) for s in (a, b)])
    before = session.account()
    with pytest.raises(CacheFull):                                   # the last chunk has no room: none of them runs
        session.step([StepEntry(a, prompt(300, 3), [0]), StepEntry(b, prompt(600, 4), [0])])
    assert session.unchanged_since(before)
    session.close(a)
    session.close(b)
    assert sorted(session.free) == list(range(16))


# ---- models that are refused --------------------------------------------------------------------------------------
def _model(window=None, stops=((0, 0), (1, 1)), embedding=None, **kw):
    from supersonic_b200.config.base import ScheduleEntry
    from supersonic_b200.parts.attention import Attention
    from supersonic_b200.parts.block import PreNormBlock
    from supersonic_b200.parts.feed_forward import SwiGLU

    def block():
        mixer, ff = Attention.__new__(Attention), SwiGLU.__new__(SwiGLU)
        vars(mixer).update(n_q=1, n_kv=1, head_dim=16, window=window, scale=1.0, w_qkv=torch.zeros((48, 16)), w_o=torch.zeros((16, 16)))
        vars(ff).update(act=None, inter=16, layout="stacked", w_gate_up=torch.zeros((32, 16)), w_down=torch.zeros((16, 16)))
        return PreNormBlock(mixer, ff, None, None, SimpleNamespace(rotary_tables=lambda: None, interleaved=False, rotary_dim=16))
    schedule = [ScheduleEntry(*stop, **(kw if i == 1 else {})) for i, stop in enumerate(stops)]
    return SimpleNamespace(device=torch.device("cpu"), dtype=torch.float32, blocks=[block(), block()], vocab_size=VOCAB, use_graphs=False,
                           spec=SimpleNamespace(schedule=schedule), step_token_budget=64, embedding=embedding, _check_positions=lambda n: None)


def test_models_that_a_session_would_run_wrongly_are_refused(monkeypatch):
    monkeypatch.setattr(int8_ops, "quantize_rows", lambda *a: None)
    Int8Session(_model(), 256)
    Int8Session(_model(window=100), 256)
    for model in (_model(before=(0, 0)), _model(writes_cache=False), _model(stops=((0, 0), (1, 0))), _model(stops=((1, 0), (0, 1))),
                  _model(embedding=SimpleNamespace(cache_need=lambda: None))):
        with pytest.raises(ValueError):
            Int8Session(model, 256)
    with pytest.raises(ValueError):                                  # a window counts positions, a cut cache has places
        Int8Session(_model(window=100), 256, budget=64)
