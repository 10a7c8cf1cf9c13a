"""How a scorer's workspace grows under calls of ever larger batches (no GPU)."""
from promptboot_amd import scores


class Recorder(scores.RowScorer):
    def __init__(self):
        self.sampler, self._own, self._reserved, self.calls = None, False, (0, 0), []

    def reserve(self, rows, vocab=0):
        self.calls.append((rows, vocab))
        self._reserved = tuple(max(a, b) for a, b in zip(self._reserved, (rows, vocab)))


def test_every_call_fits_and_few_of_them_grow():
    sc = Recorder()
    for n in range(1, 4097):
        sc._ensure(n, 151_936)
        assert sc._reserved[0] >= n and sc._reserved[1] >= 151_936
    assert len(sc.calls) <= 13
    # what was outgrown adds up to less than what is in use
    assert sum(r for r, _ in sc.calls[:-1]) < sc.calls[-1][0] <= 2 * 4096
    for n in range(151_937, 160_000):
        sc._ensure(1, n)
    assert len(sc.calls) <= 14
    assert all(r <= 8192 and v <= 2 * 151_936 for r, v in sc.calls)


def test_a_first_call_reserves_what_it_needs_and_limits_hold():
    sc = Recorder()
    sc._ensure(700, 1000)
    assert sc.calls == [(700, 1000)]
    sc._ensure(5, 900)
    assert sc.calls == [(700, 1000)]
    sc._ensure(700_000, 3_000_000)
    sc._ensure(scores.SCORE_MAX_ROWS, scores.SCORE_MAX_VOCAB)
    assert sc._reserved == (scores.SCORE_MAX_ROWS, scores.SCORE_MAX_VOCAB)
    sc._ensure(scores.SCORE_MAX_ROWS + 1, 5)  # the reservation itself refuses it
    assert sc.calls[-1][0] == scores.SCORE_MAX_ROWS + 1


def test_reservations_cover_every_pair_of_what_they_name(monkeypatch):
    """Many short rows, then few long ones: a call of many long rows does not reserve again, so both must fit."""
    asked = []

    class Lib:
        @staticmethod
        def pb_context_reserve_scores(ctx, rows, vocab, err):
            asked.append((rows, vocab))
            return 0

    class Context:
        _ctx, device = 1, 0

    monkeypatch.setattr(scores, "lib", lambda: Lib)
    sc = scores.RowScorer(sampler=Context())
    sc.reserve(1000, 100)
    sc.reserve(10, 50_000)
    sc._ensure(1000, 50_000)
    assert any(rows >= 1000 and vocab >= 50_000 for rows, vocab in asked)
    sc.reserve(5, 5)
    assert sc._reserved == (1000, 50_000)
