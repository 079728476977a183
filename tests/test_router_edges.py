"""The router on a GPU where its calls are unusual: slots without an expert before a rank whose first expert is a negative
number, groups with a single expert left, calls from several threads at once, plans made under graph capture."""
import subprocess
import sys
import threading
from pathlib import Path

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


def test_calls_from_several_threads_at_once():
    """Threads whose sorts need different amounts of shared memory, each on a stream of its own: no call fails another's."""
    shapes = [(60, 16, 1024), (20, 32, 1024), (64, 12, 700), (33, 8, 900)]      # tokens, slots, the rank's experts of 1024
    failed, plans = [], []
    for i, (T, k, local) in enumerate(shapes):
        plan, ids, _, sort = run(logits_of(i, T, 1024), k, local)
        outs = [ids, sort["sorted_tok"], sort["expert_offset"]]
        plans.append((plan, torch.cuda.Stream(), outs, [t.clone() for t in outs]))
    flat = torch.randint(0, 1000, (2000,), dtype=torch.int32, device="cuda")
    scatters = [(n, torch.empty(2000, dtype=torch.int32, device="cuda"), torch.empty(n + 1, dtype=torch.int32, device="cuda"))
                for n in (1000, 450)]
    torch.cuda.synchronize()

    def routes(plan, stream):
        for _ in range(3000):
            try:
                plan.run(stream.cuda_stream)
            except RuntimeError as e:
                failed.append(e)

    def sorts(n, tok, off, stream):
        for _ in range(3000):
            try:
                dense.native().moe_scatter(flat.data_ptr(), 2000, n, 0, tok.data_ptr(), off.data_ptr(), None, stream.cuda_stream)
            except RuntimeError as e:
                failed.append(e)

    threads = [threading.Thread(target=routes, args=p[:2]) for p in plans]
    threads += [threading.Thread(target=sorts, args=(*o, torch.cuda.Stream())) for o in scatters]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed, (len(failed), failed[0])
    for _, _, outs, olds in plans:
        assert all(torch.equal(t, old) for t, old in zip(outs, olds))


@pytest.mark.parametrize("local", [12287, 12288, 16384])
@pytest.mark.parametrize("T", [40, 300])
def test_the_largest_ranks(T, local):
    """Counts of a rank's experts past the 48 KB of shared memory that a kernel has without asking."""
    base = 100 - local                      # its last experts are the ones there are
    _, ids, _, sort = run(logits_of(T, T, 100), 8, local, base)
    tok, off = sorted_by_definition(ids.cpu().numpy(), local, base)
    assert np.array_equal(sort["expert_offset"].cpu().numpy(), off)
    assert np.array_equal(sort["sorted_tok"].cpu().numpy(), tok)


def equal_sort(ids, local, base, tok, off):
    for want, got in zip(sorted_by_definition(ids.cpu().numpy(), local, base), (tok, off)):
        assert np.array_equal(got.cpu().numpy(), want)


def scatter_of_nearly_48_kilobytes():
    native, stream = dense.native(), torch.cuda.current_stream().cuda_stream
    for T in (20, 32):
        for local in (371, 372, 373):
            ids = torch.randint(-1, 400, (T, 8), generator=torch.Generator().manual_seed(T), dtype=torch.int32).cuda()
            tok, off = (torch.empty(n, dtype=torch.int32, device="cuda") for n in (T * 8, local + 1))
            native.moe_scatter(ids.data_ptr(), T * 8, local, 0, tok.data_ptr(), off.data_ptr(), None, stream)
            equal_sort(ids, local, 0, tok, off)
            l, w = logits_of(T, T, 400), torch.empty((T, 8), device="cuda")
            native.router_scatter(l.data_ptr(), T, 400, 8, ids.data_ptr(), w.data_ptr(), local, 0, tok.data_ptr(), off.data_ptr(),
                                  None, stream)
            equal_sort(ids, local, 0, tok, off)


def router_of_nearly_48_kilobytes():
    for local in (992, 993, 994, 995):
        _, ids, _, sort = run(logits_of(1, 44, 1000), 8, local, 3)
        equal_sort(ids, local, 3, sort["sorted_tok"], sort["expert_offset"])


@pytest.mark.parametrize("what", ["scatter", "router"])
def test_a_sort_of_nearly_48_kilobytes(what):
    """Tables of 48 KB less than a kernel's static arrays. In a process of its own: a kernel keeps the limit that a larger call
    has set."""
    code = f"import conftest, test_router_edges as t; t.{what}_of_nearly_48_kilobytes()"
    subprocess.run([sys.executable, "-c", code], cwd=Path(__file__).parent, check=True, timeout=300)


@pytest.mark.parametrize("T", [8, 200, 700])
def test_a_plan_made_under_capture(T):
    """As other plans can be: in one launch, with the one-block sort, and with the sort that has a work buffer."""
    l = logits_of(1, T, 256)
    _, want, _, want_sort = run(l, 8, 256)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan, ids, _, sort = run(l, 8, 256)
    for _ in range(2):
        graph.replay()
        assert torch.equal(ids, want)
        assert all(torch.equal(sort[n], want_sort[n]) for n in ("sorted_tok", "expert_offset"))
        ids.zero_()


NONE = float("-inf")
LONE = [                                                        # c by group, groups kept, the chosen experts
    ([[.875], [.5, .25], [], [.125, .1875]], 1, [0, -1, -1]),
    ([[.875], [.5, .25], [], [.125, .1875]], 2, [0, 4, 5]),
    ([[], [.5], [], [.0625, .125]], 3, [4, 13, 12]),
    ([[.75 + 2.0 ** -22], [.5, .25]], 1, [0, -1, -1]),          # sums that the 64-bit scores tell apart
    ([[.75 - 2.0 ** -22], [.5, .25]], 1, [4, 5, -1]),
    ([[.75], [.5, .25]], 1, [0, -1, -1]),                       # and equal ones
    ([[.5, .25], [.75]], 1, [0, 1, -1]),
    ([[-.125], [-.0625, -.125]], 1, [0, -1, -1])]


@pytest.mark.parametrize("by", ["logit", "bias"])
@pytest.mark.parametrize("c,keep,want", LONE)
@pytest.mark.parametrize("T", [3, 300])
def test_a_group_with_one_expert_left_is_ranked_by_it(T, c, keep, want, by):
    """Masked experts, by their logit or by their bias, are left out of their group's sum of two. Sigmoid's s is 1/2 throughout."""
    c = torch.tensor([(g + [NONE] * 4)[:4] for g in (c + [[]] * 4)[:4]]).reshape(16)
    row, bias = torch.zeros(16), c - 0.5
    if by == "logit":
        row, bias = torch.where(c == NONE, NONE, row), bias.nan_to_num(neginf=0.25)
    logits = row.expand(T, 16).contiguous().cuda()
    _, ids, w, _ = run(logits, 3, score="sigmoid", bias=bias.cuda(), groups=4, keep_groups=keep, group_top=2)
    assert ids.tolist() == [want] * T
    assert w.tolist() == [[0.0 if e < 0 else 0.5 for e in want]] * T


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_an_expert_masked_by_its_bias_still_counts_in_the_softmax(score):
    """Its logit does; a masked logit does not."""
    l, bias = torch.zeros((2, 8), device="cuda"), torch.zeros(8, device="cuda")
    bias[:4] = NONE
    l[1, [0, 7]] = NONE
    _, ids, w, _ = run(l, 4, score=score, bias=bias)
    assert ids.tolist() == [[4, 5, 6, 7], [4, 5, 6, -1]]
    of = [2.0 ** -3, 1 / 6] if score == "softmax" else [0.5, 0.5]
    want = torch.tensor([[of[0]] * 4, [of[1]] * 3 + [0.0]], dtype=torch.float64)
    assert ((w.cpu().double() - want).abs() <= 2.0 ** -24 * 88 * want).all()      # test_router's tolerance, z the largest logit
