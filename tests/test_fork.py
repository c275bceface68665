"""DecodeStack's forks without a GPU: whose blocks a table holds, and what each call refuses or copies. The pool is a tensor of row marks, a step
writes the mark of its token where the table points."""
import pytest
import torch

from embla_metal_b200 import stack as stk

PAGES = 4


class _Pool:
    def __init__(self, blocks):
        self.rows = torch.full((blocks, 128), -1)


class _Ctx:
    def copy_blocks(self, pool, src, dst, rows=None):
        for i in range(src.numel()):
            n = 128 if rows is None else int(rows[i])
            pool.rows[int(dst[i]), :n] = pool.rows[int(src[i]), :n]


def _stack(batch):
    st = stk.DecodeStack.__new__(stk.DecodeStack)
    st.batch, st.npages, st.max_context, st.max_seq_len = batch, PAGES, PAGES * 128, PAGES * 128
    st.ctx, st.full_pool, st.sparse_pool, st.rings = _Ctx(), _Pool(batch * PAGES), None, []
    st.table = torch.arange(batch * PAGES, dtype=torch.int32).view(batch, PAGES).contiguous()
    st._owner, st._standing = [[b] * PAGES for b in range(batch)], []
    st.pos, st.seq_lens = torch.zeros(batch, dtype=torch.int32), torch.zeros(batch, dtype=torch.int32)
    st.qkv = st.o = torch.zeros(1, batch, 1)
    st.handle = None
    return st


def _step(st, marks):
    """What a step writes: the token's row of every sequence, all of them before any is read."""
    st._step_struct()
    at = [(int(st.table[b, int(st.pos[b]) // 128]), int(st.pos[b]) % 128) for b in range(st.batch)]
    assert len(set(at)) == st.batch, "two sequences write one row"
    for (block, row), m in zip(at, marks):
        st.full_pool.rows[block, row] = m


def _rows(st, b, n):
    return st.full_pool.rows[st.table[b].long()].flatten()[:n].tolist()


def _fill(st, n):
    """n steps, sequence b marking position t with 1000 b + t."""
    for t in range(n):
        st.set_positions(t)
        _step(st, [1000 * b + t for b in range(st.batch)])


@pytest.mark.parametrize("n", [1, 127, 128, 129, 256, 300])
@pytest.mark.parametrize("ahead", [False, True])
def test_fork_then_steps_keep_the_sequences_apart(n, ahead):
    """Forked behind a step that wrote position n - 1, or with the positions moved on to it already: the next steps, with or without
    set_positions, write rows of each sequence's own."""
    st = _stack(3)
    _fill(st, n - 1 if ahead else n)
    if ahead:
        st.set_positions(n - 1)
    st.fork(0, 2)
    _step(st, [1, 2, 3])                                   # no set_positions: position n - 1 (again)
    for i in range(3):
        st.set_positions(n + i)
        _step(st, [10 + i, 20 + i, 30 + i])
    head = list(range(n - 1))
    assert _rows(st, 0, n + 3) == head + [1, 10, 11, 12]
    assert _rows(st, 2, n + 3) == head + [3, 30, 31, 32]
    assert _rows(st, 1, n + 3) == [1000 + t for t in head] + [2, 20, 21, 22]


@pytest.mark.parametrize("who", [0, 1, 2])
def test_a_chain_of_forks_on_the_last_row(who):
    """0 -> 1 -> 2, all at 256 keys; one of them writes position 255 once more, the others go on behind it."""
    st = _stack(3)
    _fill(st, 256)
    st.fork(0, 1)
    st.fork(1, 2)
    at = [256] * 3
    at[who] = 255
    st.set_positions(at)
    _step(st, [1, 2, 3])
    for b in range(3):
        assert _rows(st, b, at[b] + 1) == list(range(at[b])) + [b + 1]
    assert all(int(st.table[b, 0]) == 0 for b in range(3))


def test_moved_on_positions_stay_shared_and_are_refused_later():
    st = _stack(2)
    _fill(st, 128)
    st.fork(0, 1)
    st.set_positions(128)
    assert int(st.table[1, 0]) == 0
    for p in ([127, 128], [128, 127]):
        with pytest.raises(ValueError):
            st.set_positions(p)
    with pytest.raises(ValueError):
        st.restart(0)
    st.restart(1)
    st.set_positions([127, 0])
    assert int(st.table[1, 0]) == PAGES


def test_restart_and_another_fork_forget_the_first():
    st = _stack(3)
    _fill(st, 128)
    st.fork(0, 1)
    st.restart(1)
    _step(st, [1, 2, 3])
    assert _rows(st, 0, 128)[-1] == 1 and _rows(st, 1, 1) == [2]
    st.set_positions([127, 100, 127])
    st.fork(0, 1)
    st.fork(2, 1)                                          # dst again, of another source
    _step(st, [4, 5, 6])
    assert _rows(st, 0, 128)[-1] == 4 and _rows(st, 1, 128) == [2000 + t for t in range(127)] + [5] and _rows(st, 2, 128)[-1] == 6


def _chunk(st, monkeypatch, pos0, T, mark=0, **kw):
    """prefill_chunk with a library that writes the rows' marks: 1000 b + position + mark."""
    class Lib:
        @staticmethod
        def embla_stack_prefill_chunk(handle, ck, stream):
            for b, p0 in enumerate(pos0):
                for t in range(p0, p0 + T):
                    st.full_pool.rows[int(st.table[b, t // 128]), t % 128] = 1000 * b + t + mark
            return 0
    monkeypatch.setattr(stk.attn, "lib", lambda: Lib)
    monkeypatch.setattr(stk.attn, "_stream", lambda: None)
    st.kinds = [stk.FULL]
    x = torch.zeros(1, st.batch, T, 1)
    st.prefill_chunk(x, x, torch.tensor(pos0, dtype=torch.int32), **kw)


@pytest.mark.parametrize("n", [1, 127, 128, 129, 256, 300])
@pytest.mark.parametrize("used", [0, 400])
@pytest.mark.parametrize("positions", [False, True])
def test_fork_after_a_chunk_has_the_prompt(n, used, positions, monkeypatch):
    """A prompt of n tokens, on a new stack or behind other work, forked; the next tokens are those at n, whether or not the caller says so."""
    st = _stack(3)
    if used:
        _fill(st, used)
    _chunk(st, monkeypatch, [0, 0, 0], n, max_seq_len=n)
    st.fork(0, 2)
    for i in range(3):
        if i or positions:
            st.set_positions(n + i)
        _step(st, [10 + i, 20 + i, 30 + i])
    head = list(range(n))
    assert _rows(st, 0, n + 3) == head + [10, 11, 12]
    assert _rows(st, 2, n + 3) == head + [30, 31, 32]
    assert _rows(st, 1, n + 3) == [1000 + t for t in head] + [20, 21, 22]


def test_positions_behind_a_chunk(monkeypatch):
    st = _stack(2)
    st.set_positions([3, 9])
    _chunk(st, monkeypatch, [4, 200], 100, max_seq_len=300)
    assert st.pos.tolist() == [104, 300] and st.seq_lens.tolist() == [105, 301] and st.max_seq_len == 301
    _chunk(st, monkeypatch, [0, PAGES * 128 - 100], 100, max_seq_len=PAGES * 128)   # the second sequence's context is full
    assert st.pos.tolist() == [100, PAGES * 128 - 1] and st.seq_lens.tolist() == [101, PAGES * 128]
    assert st.max_seq_len == PAGES * 128
    st.set_positions([1, 1])
    _chunk(st, monkeypatch, [0, 0], 100)                   # no bound given
    assert st.max_seq_len == PAGES * 128


def test_a_chunk_does_not_write_shared_blocks(monkeypatch):
    st = _stack(3)
    _chunk(st, monkeypatch, [0, 0, 0], 300, max_seq_len=300)
    st.fork(0, 2)
    before, at = st.full_pool.rows.clone(), st.pos.tolist()
    for pos0 in ([0, 0, 300], [300, 0, 255], [255, 300, 256], [0, 0, 0]):
        with pytest.raises(ValueError):
            _chunk(st, monkeypatch, pos0, 100, mark=5, max_seq_len=400)
    assert torch.equal(st.full_pool.rows, before) and st.pos.tolist() == at
    _chunk(st, monkeypatch, [256, 0, 300], 100, mark=5, max_seq_len=400)   # behind them
    head = list(range(256))
    assert _rows(st, 0, 356) == head + [t + 5 for t in range(256, 356)]
    assert _rows(st, 2, 400) == head + list(range(256, 300)) + [2000 + t + 5 for t in range(300, 400)]
    st.restart(2)                                          # a new prompt for all of them
    _chunk(st, monkeypatch, [0, 0, 0], 10, mark=7, max_seq_len=10)
    assert [_rows(st, b, 10) for b in range(3)] == [[1000 * b + t + 7 for t in range(10)] for b in range(3)]


def test_a_chunk_from_the_last_row_of_a_shared_block(monkeypatch):
    st = _stack(2)
    _fill(st, 256)
    st.fork(0, 1)
    _chunk(st, monkeypatch, [255, 255], 3, mark=5, max_seq_len=258)
    assert _rows(st, 0, 258) == list(range(255)) + [260, 261, 262]
    assert _rows(st, 1, 258) == list(range(255)) + [1260, 1261, 1262]


@pytest.mark.parametrize("pos0", [torch.zeros(2), torch.zeros(2, dtype=torch.int64), torch.zeros(1, dtype=torch.int32),
                                  torch.zeros(2, dtype=torch.int32, device="meta")])
def test_a_chunk_refuses_positions_that_are_not_the_stack_s(pos0, monkeypatch):
    st = _stack(2)
    st.kinds = [stk.FULL]
    called = []
    monkeypatch.setattr(stk.attn, "lib", lambda: called.append(1))
    with pytest.raises(ValueError):
        st.prefill_chunk(torch.zeros(1, 2, 3, 1), torch.zeros(1, 2, 3, 1), pos0)
    assert not called and st.pos.tolist() == [0, 0]


@pytest.mark.parametrize("seed", range(60))
def test_random_forks_chunks_and_steps(seed, monkeypatch):
    """Any order of calls: what each sequence's table holds is what that sequence wrote, or has from where it was forked; a call that is refused
    changes nothing."""
    import random
    rng = random.Random(seed)
    B, cap = 4, PAGES * 128
    st = _stack(B)
    st.set_positions(0)
    rows = [[] for _ in range(B)]                          # what sequence b has written: its positions 0 .. len - 1
    near = lambda n: min(cap - 3, max(0, rng.choice([n, n, n, n - 1, n // 128 * 128 - 1, n // 128 * 128, rng.randint(0, n)])))
    done = 0
    for turn in range(150):
        kind = rng.choice(["step", "step", "chunk", "fork", "fork", "restart"])
        if kind == "step":
            at = [near(len(r)) for r in rows]
            if rng.random() < 0.7:
                try:
                    st.set_positions(at)
                except ValueError:
                    assert any(st._shared(b) for b in range(B))
                    continue
            at = st.pos.tolist()
            if any(p > len(r) for p, r in zip(at, rows)):
                continue                                   # (positions behind what is there: not after a refusal)
            marks = [10 ** 6 * turn + b for b in range(B)]
            _step(st, marks)
            for b, p in enumerate(at):
                rows[b][p:] = [marks[b]]
        elif kind == "chunk":
            T = rng.choice([1, 2, 100, 128, 129])
            at = [min(near(len(r)), cap - T) for r in rows]
            try:
                _chunk(st, monkeypatch, at, T, mark=10 ** 6 * turn, max_seq_len=max(at) + T)
            except ValueError:
                assert any(st._shared(b) for b in range(B))
                continue
            for b, p in enumerate(at):
                rows[b][p:] = [1000 * b + t + 10 ** 6 * turn for t in range(p, p + T)]
        elif kind == "fork":
            src, dst = rng.sample(range(B), 2)
            n = int(st.seq_lens[src])
            if n > len(rows[src]) + 1:
                continue
            try:
                st.fork(src, dst)
            except ValueError:
                assert st._lent_to(dst)
                continue
            rows[dst] = rows[src][:n]
        else:
            b = rng.randrange(B)
            try:
                st.restart(b)
            except ValueError:
                assert st._lent_to(b)
                continue
            rows[b] = []
        done += 1
        for b in range(B):
            assert _rows(st, b, len(rows[b])) == rows[b], (turn, kind, b)
    assert done > 40
