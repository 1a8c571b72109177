"""The tree rounds' host side: what they refuse, and what a failed round leaves (no GPU needed)."""
from types import SimpleNamespace

import pytest
import torch

import spec.tree as rounds


class Cache:
    device = torch.device("cpu")

    def add(self, seq_id):
        pass

    def free(self, seq_id):
        pass

    def truncate(self, seq_id, length):
        pass


class Drafter:
    def __init__(self):
        self.proposed = 0

    def prefill(self, seq_ids, prompts):
        pass

    def propose(self, seq_ids, contexts):
        self.proposed += 1
        return torch.tensor([[c[-1], 4, 5] for c in contexts]), torch.tensor([[-1, 0, 1]])

    def rollback(self, seq_id, keep):
        pass

    def release(self, seq_id):
        pass


def run_rounds(monkeypatch, firsts, verdicts):
    """generate_tree of two prompts whose first tokens and rounds' verdicts [N + 1, B] are given."""
    verdicts = iter(verdicts)
    monkeypatch.setattr(rounds, "run", lambda *a: torch.zeros(2, 9))
    monkeypatch.setattr(rounds, "draw", lambda *a: torch.tensor(firsts))
    monkeypatch.setattr(rounds, "verify_tree", lambda *a: torch.tensor(next(verdicts)))
    drafter = Drafter()
    return drafter, lambda: rounds.generate_tree(None, Cache(), drafter, [[1, 2], [3]], 6)


GOOD = [[2, 0], [7, 8], [4, -1], [5, -1]]  # three tokens for one row, one for the other


def test_rounds_settle(monkeypatch):
    _, go = run_rounds(monkeypatch, [6, 6], [GOOD, [[1, 2], [8, 8], [4, 4], [-1, 5]], [[2], [7], [4], [5]]])
    out, stats = go()
    assert out == [[6, 4, 5, 7, 4, 8], [6, 8, 4, 5, 8, 4]] and stats.rounds == 3


def test_a_first_token_that_is_none_ends_the_call(monkeypatch):
    drafter, go = run_rounds(monkeypatch, [6, -1], [])
    with pytest.raises(RuntimeError, match="seq 1.*no token"):
        go()
    assert drafter.proposed == 0


@pytest.mark.parametrize("bad", [[[2, 0], [7, -1], [4, -1], [5, -1]], [[2, -1], [7, 8], [4, -1], [5, -1]]])
def test_a_round_without_a_token_ends_the_call(monkeypatch, bad):
    """A row whose logits are no numbers (token -1), and one whose commit found no slot (n = -1)."""
    drafter, go = run_rounds(monkeypatch, [6, 6], [GOOD, bad])
    with pytest.raises(RuntimeError, match="seq 1.*no token"):
        go()
    assert drafter.proposed == 2  # the second round's, and none after it


def test_a_drafter_has_a_level_at_least():
    with pytest.raises(ValueError, match="level"):
        rounds.ModelTree(None, SimpleNamespace(device=torch.device("cpu")), [])
    with pytest.raises(ValueError, match="child"):
        rounds.ModelTree(None, SimpleNamespace(device=torch.device("cpu")), [2, 0])
    assert rounds.tree_shape([]).tolist() == [[-1]]  # a tree of node 0 alone can be verified


def test_a_sequence_has_one_row_of_a_verify():
    cache = SimpleNamespace(length=lambda s: 1, device=torch.device("cpu"))
    with pytest.raises(ValueError, match="once"):
        rounds.verify_tree(None, cache, [3, 3], [[1, 2], [1, 2]], torch.tensor([[2, 5], [2, 6]]), torch.tensor([[-1, 0]]),
                           torch.zeros(2, 2))
