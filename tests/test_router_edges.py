"""The router on a GPU where its calls are unusual: slots without an expert before a rank whose first expert is a negative
number, groups with a single expert left, calls from several threads at once, plans made under graph capture."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from exl3b200 import dense  # noqa: E402
from test_router import gpu, logits_of, run  # noqa: E402, F401


def sorted_by_definition(ids, local, base):
    """(sorted_tok, expert_offset): a stable sort; negative ids, and those outside the rank's, are no expert's."""
    flat = ids.reshape(-1).astype(np.int64)
    e = np.where((flat >= 0) & (flat >= base) & (flat < base + local), flat - base, local)
    off = np.concatenate(([0], np.cumsum(np.bincount(e, minlength=local + 1)[:local])))
    order = np.argsort(e, kind="stable")
    return np.where(np.arange(len(flat)) < off[-1], order, -1), off


@pytest.mark.parametrize("T", [5, 12, 90, 700])
@pytest.mark.parametrize("local,base", [(400, -300), (1500, -1000), (64, 0), (20, 7)])
def test_slots_without_an_expert_are_nobodys(T, local, base):
    """Three experts for eight slots; in one launch with the sort, in its one-block form, and in its three launches."""
    l = torch.full((T, 64), -torch.inf, device="cuda")
    l[:, [3, 9, 40]] = logits_of(T, T, 3)
    _, ids, w, sort = run(l, 8, local, base)
    got = ids.cpu().numpy()
    assert (got[:, 3:] == -1).all() and (np.sort(got[:, :3]) == [3, 9, 40]).all() and (w[:, 3:] == 0).all()
    tok, off = sorted_by_definition(got, local, base)
    assert np.array_equal(sort["expert_offset"].cpu().numpy(), off)
    assert np.array_equal(sort["sorted_tok"].cpu().numpy(), tok)
