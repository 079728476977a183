"""router on a GPU against a plain implementation in 64 bits.

ids, and the sort, are compared exactly: choices follow the logits, or 64-bit scores. Tolerance of the weights, relative, in
units of 2^-24: the difference z - m of two f32 numbers is off by half a unit of itself, which the exponential makes |z - m|
units at most; expf by 4 (2 units in the last place); the softmax's denominator by as much again (its terms' errors weighted by
the terms: the largest |d| e^-|d| is 0.37, and expf's 4) and by one a term added, at most 64 in a lane and 5 across them;
division, scale and sigmoid's sum one each. |z - m| + 88 covers them."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from exl3b200 import dense  # noqa: E402

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    torch.cuda.set_device(0)
    yield
    torch.cuda.synchronize()
    assert dense.native().read_error() == 0


def plain(logits, top_k, score="softmax", bias=None, groups=1, keep_groups=1, group_top=1, renorm=False, scale=1.0):
    """(ids, w, tolerance of w) in numpy's 64 bits."""
    l = logits.double().cpu().numpy().copy()
    b = np.zeros(l.shape[1]) if bias is None else bias.double().cpu().numpy()
    T, E = l.shape
    l[np.isnan(l)] = -np.inf
    l = np.minimum(l, float(np.finfo(np.float32).max))
    ids, w, tol = np.full((T, top_k), -1, np.int64), np.zeros((T, top_k)), np.zeros((T, top_k))
    for t in range(T):
        with np.errstate(over="ignore", invalid="ignore"):
            top = l[t].max()
            if score == "softmax":
                s = np.exp(l[t] - top) if top > -np.inf else np.zeros(E)
                s = s / s.sum() if top > -np.inf else s
            else:
                s = 1 / (1 + np.exp(-l[t]))
            wide = bias is not None or (keep_groups < groups and group_top == 2)
            c = s + b if wide else l[t].copy()
        c[np.isneginf(l[t]) | np.isnan(c)] = -np.inf
        if keep_groups < groups:
            by = -np.sort(-c.reshape(groups, -1), axis=1)[:, :group_top]
            best = np.where(np.isneginf(by), 0, by).sum(1)
            best[np.isneginf(by[:, 0])] = -np.inf
            kept = np.argsort(-best, kind="stable")[:keep_groups]
            c[~np.isin(np.arange(E) // (E // groups), kept)] = -np.inf
        order = [e for e in np.argsort(-c, kind="stable")[:top_k] if c[e] > -np.inf]
        if not order:
            continue
        z = l[t, order]
        most = z.max()
        if renorm and (score == "softmax" or most < -20):
            v = np.exp(z - most)
        else:
            v = s[order]
        v = v / v.sum() if renorm else v
        ids[t, :len(order)], w[t, :len(order)] = order, v * scale
        d = np.abs(z - (top if score == "softmax" and not renorm else most)) if score == "softmax" or most < -20 else 0 * z
        tol[t, :len(order)] = np.abs(v * scale) * 2.0 ** -24 * (d + 88)
    return ids, w, tol + 2.0 ** -149 * max(1.0, abs(scale))


def run(logits, top_k, local=None, base=0, **kw):
    T, E = logits.shape
    ids = torch.full((T, top_k), -7, dtype=torch.int32, device="cuda")
    w = torch.full((T, top_k), -7.0, device="cuda")
    sort = {}
    if local:
        sort = dict(sorted_tok=torch.full((T * top_k,), -7, dtype=torch.int32, device="cuda"),
                    expert_offset=torch.full((local + 1,), -7, dtype=torch.int32, device="cuda"), expert_base=base)
    plan = dense.Router(logits=logits, top_k=top_k, ids=ids, w=w, **kw, **sort)
    plan.run()
    return plan, ids, w, sort


def check(logits, top_k, local=None, base=0, **kw):
    _, ids, w, sort = run(logits, top_k, local, base, **kw)
    want, want_w, tol = plain(logits, top_k, **kw)
    got = ids.cpu().numpy()
    assert np.array_equal(got, want), np.argwhere(got != want)[:5]
    err = np.abs(w.double().cpu().numpy() - want_w)
    assert (err <= tol).all(), (err / tol).max()
    if local:
        flat = want.reshape(-1)
        e = np.where((flat >= base) & (flat < base + local), flat - base, local)
        order = np.argsort(e, kind="stable")
        off = np.concatenate(([0], np.cumsum(np.bincount(e, minlength=local + 1)[:local])))
        order = np.where(np.arange(len(flat)) < off[-1], order, -1)
        assert np.array_equal(sort["expert_offset"].cpu().numpy(), off)
        assert np.array_equal(sort["sorted_tok"].cpu().numpy(), order)


def logits_of(seed, T, E, dtype=F32, scale=1.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (scale * torch.randn((T, E), generator=g, device="cuda")).to(dtype)


def bias_of(seed, E, scale=0.1):
    return scale * torch.randn(E, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("renorm", [False, True])
@pytest.mark.parametrize("E,k,groups,keep,top", [(512, 10, 1, 1, 1), (256, 8, 8, 4, 2), (160, 6, 8, 3, 1), (96, 4, 3, 2, 2),
                                                 (1, 1, 1, 1, 1), (7, 7, 1, 1, 1), (64, 1, 32, 5, 2), (1000, 32, 1, 1, 1),
                                                 (2048, 16, 16, 7, 2), (45, 5, 5, 2, 2), (33, 20, 1, 1, 2)])
def test_scores_biases_and_groups(E, k, groups, keep, top, renorm, bias, score):
    kw = dict(score=score, groups=groups, keep_groups=keep, group_top=top, renorm=renorm, scale=2.5 if renorm else 1.0)
    check(logits_of(E + k, 37, E), k, bias=bias_of(E, E) if bias else None, **kw)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("T", [1, 2, 31, 32, 33, 300, 2500])
def test_types_and_token_counts_with_the_sort(T, dtype):
    """16-bit logits hold equal ones."""
    kw = dict(score="sigmoid", groups=8, keep_groups=4, group_top=2, renorm=True, scale=2.5)
    check(logits_of(T, T, 256, dtype), 8, local=256, bias=bias_of(1, 256), **kw)
    check(logits_of(T + 1, T, 512, dtype), 10, local=512)


@pytest.mark.parametrize("T", [3, 4, 5, 16, 17, 28, 29, 48, 63, 64, 65, 97, 127, 128, 129])
@pytest.mark.parametrize("E,k,local,base", [(512, 10, 512, 0), (256, 8, 256, 0), (40, 5, 40, 0), (1024, 32, 1024, 0),
                                            (2048, 16, 1024, 512), (64, 32, 8, 30)])
def test_the_sort_in_one_launch_and_in_its_own(T, E, k, local, base):
    """A CTA for each four tokens, up to eight of them with sixteen; by the size of the sort's table, launches of its own."""
    check(logits_of(T, T, E), k, local=local, base=base, renorm=True)
    check(logits_of(T, T, E, BF16), k, local=local, base=base, score="sigmoid", bias=bias_of(T, E))


def test_the_sort_over_a_ranks_experts():
    for T in (20, 700):
        check(logits_of(T, T, 512), 10, local=128, base=256, renorm=True)
        check(logits_of(T, T, 512), 10, local=1500, base=-1000, renorm=True)


@pytest.mark.parametrize("groups,keep,top", [(1, 1, 1), (8, 3, 1), (8, 3, 2)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
def test_masked_experts_and_rows_with_nothing(bias, score, groups, keep, top):
    l = logits_of(3, 12, 64)
    l[0] = -torch.inf
    l[1] = torch.nan
    l[2, 5:] = -torch.inf                                       # five left, one group
    l[3, torch.arange(64, device="cuda") % 8 != 3] = -torch.inf    # one a group
    l[4, ::2] = torch.nan
    l[5, [7, 40]] = torch.inf
    l[6] = torch.inf
    l[7, 1:] = -3e38
    l[8] = 3.4e38
    l[9, 10] = 200.0
    l[10] = -500.0
    b = bias_of(4, 64) if bias else None
    if bias:
        b[8:12] = -torch.inf
        b[20] = torch.nan
        b[30] = torch.inf
    for renorm in (False, True):
        check(l, 8, local=64, score=score, bias=b, groups=groups, keep_groups=keep, group_top=top, renorm=renorm)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_equal_scores_go_to_the_lower_expert(score):
    for v in (0.0, -0.0, 3.0):
        l = torch.full((40, 200), v, device="cuda")
        l[::2, ::3] = -v
        check(l, 9, score=score, renorm=True)
        check(l, 9, score=score, bias=torch.zeros(200, device="cuda"), groups=4, keep_groups=2, group_top=2)


def test_scores_that_differ_by_less_than_their_rounding():
    """Biases that bring every c to within f32's last place of 0.7: the order is that of 64 bits."""
    l = logits_of(11, 400, 256)
    one = l[:1].expand(400, 256).contiguous()
    b = (0.7 - 1 / (1 + torch.exp(-one[0].double()))).float()
    check(one, 8, score="sigmoid", bias=b, groups=8, keep_groups=4, group_top=2, renorm=True)
    s = torch.softmax(one[0].double(), 0)
    check(one, 8, score="softmax", bias=(0.7 - s).float(), groups=8, keep_groups=4, group_top=2)
    check(l, 8, score="sigmoid", bias=b)


@pytest.mark.parametrize("E,k,groups,keep", [(40, 5, 1, 1), (256, 8, 8, 4), (512, 10, 16, 5), (1024, 10, 4, 2), (2048, 16, 32, 9)])
@pytest.mark.parametrize("gap", [0.0, 2.0 ** -24, 2.0 ** -20, 2.0 ** -16])
def test_neighbours_among_the_chosen(E, k, groups, keep, gap):
    """Scores in pairs that are equal or next to equal, at every place of a lane and across lanes and groups."""
    g = torch.Generator(device="cuda").manual_seed(E + groups)
    half = torch.randn((60, E // 2), generator=g, device="cuda")
    l = torch.cat((half, half * (1 + gap)), 1)[:, torch.randperm(E, generator=g, device="cuda")].contiguous()
    b = torch.zeros(E, device="cuda")
    for kw in (dict(), dict(score="sigmoid", bias=b), dict(score="softmax", bias=b + 0.25),
               dict(score="sigmoid", groups=groups, keep_groups=keep, group_top=2), dict(groups=groups, keep_groups=keep)):
        check(l, k, renorm=True, **kw)
        check(l.to(BF16), k, **kw)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_infinity_is_above_the_largest_number(dtype):
    l = logits_of(8, 3, 64, dtype)
    l[0, 9], l[0, 40] = torch.finfo(dtype).max, torch.inf
    l[1, 40], l[1, 9] = torch.finfo(dtype).max, torch.inf
    l[2, 5], l[2, 6], l[2, 7] = torch.finfo(dtype).min, 0.0, -0.0
    if dtype != F32:                    # in f32 it is the largest number
        check(l, 8)
    check(l, 32, score="sigmoid", bias=torch.zeros(64, device="cuda"))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strided_logits_and_neighbours_left_alone(dtype):
    big = torch.full((21, 700), 9.0, dtype=dtype, device="cuda")
    big[:, 3:163] = logits_of(5, 21, 160, dtype)
    check(big[:, 3:163], 6, score="sigmoid", bias=bias_of(6, 160), groups=8, keep_groups=3, group_top=2, local=160)
    ids = torch.full((23, 6), -7, dtype=torch.int32, device="cuda")
    w = torch.full((23, 6), -7.0, device="cuda")
    dense.Router(logits=big[:, 3:163], top_k=6, ids=ids[1:22], w=w[1:22]).run()
    assert (ids[[0, 22]] == -7).all() and (w[[0, 22]] == -7).all() and (ids[1:22] >= 0).all()


def test_no_tokens():
    _, ids, w, sort = run(torch.empty((0, 64), device="cuda"), 4, local=64)
    assert (sort["expert_offset"] == 0).all()


def test_captured_replayed_and_on_another_stream():
    """A plan's run in a graph, replayed over new logits; and on a side stream."""
    kw = dict(score="sigmoid", bias=bias_of(1, 256), groups=8, keep_groups=4, group_top=2, renorm=True)
    for T in (8, 500):
        l = logits_of(1, T, 256)
        plan, ids, w, sort = run(l, 8, local=256, **kw)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            plan.run()
        for seed in (2, 3):
            l.copy_(logits_of(seed, T, 256))
            graph.replay()
            want = plain(l, 8, **kw)
            assert np.array_equal(ids.cpu().numpy(), want[0])
            flat = want[0].reshape(-1)
            assert np.array_equal(sort["sorted_tok"].cpu().numpy(), np.argsort(flat, kind="stable"))
        l.copy_(logits_of(4, T, 256))
        side.wait_stream(torch.cuda.current_stream())
        plan.run(side.cuda_stream)
        side.synchronize()
        assert np.array_equal(ids.cpu().numpy(), plain(l, 8, **kw)[0])


def test_the_softmax_router_agrees_with_router_topk():
    l = logits_of(9, 100, 512)
    _, ids, w, _ = run(l, 10)
    old_ids, old_w = torch.empty_like(ids), torch.empty_like(w)
    dense.native().router_topk(l.data_ptr(), 100, 512, 10, old_ids.data_ptr(), old_w.data_ptr(),
                               torch.cuda.current_stream().cuda_stream)
    assert torch.equal(ids, old_ids)
    assert torch.allclose(w, old_w, rtol=2.0 ** -17, atol=0)    # both within (|z - m| + 88) 2^-24, |z - m| < 20
