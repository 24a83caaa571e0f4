"""GPU: policy.action_logprobs (csrc/ckr_logprobs.hip) against its definition in float64: sizes from one action to wide odd rows, three types,
masks that leave nothing, ties, values that are not finite, strides and alignments, given actions more than once, gradients against
the formula and against differences, other streams, graph replays.

Tolerances.  u = 2^-24.  A term exp(it d) of S carries the rounding of d, of it d log2(e) and of the exponential: (2 |it d| + 4) u relative;
terms that matter have |it d| <= 16 + ln V.  A sum over V terms is taken by 64 lanes (or more), each V / 64 terms in order, and joined in a few
steps: V / 64 + 16 roundings at most.  So S and the entropy's second sum are within B = (V / 64 + 2 (16 + ln V) + 32) u relative, ln S within
B absolute (plus a rounding of ln S), log p = it d - ln S within B + 4 u |log p| + 4 u ln V; H = ln S - it D / S within B (1 + 2 (ln S + H))."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def bound(v):
    return (v / 64 + 2 * (16 + math.log(v)) + 32) * U


def dark(words):
    """bool [n, 512] from legal-move words, square by square (Checkers.py:434)."""
    out = torch.zeros(words.shape[0], 512, dtype=torch.bool)
    w = words.cpu().tolist()
    for i, row in enumerate(w):
        for layer in range(8):
            for s in range(32):
                if (row[layer] & 0xFFFFFFFF) >> s & 1:
                    x = s // 4
                    out[i, 64 * layer + 8 * x + 2 * (s % 4) + (1 - x % 2)] = True
    return out.cuda()


def reference(x, allowed, actions, top, temperature):
    """float64; x [n, v], allowed bool [n, v], actions [n, k]."""
    x = x.double()
    ok = allowed & ~torch.isneginf(x)
    z = torch.where(ok, x / temperature, -math.inf)
    some = ok.any(1, keepdim=True)
    m = torch.where(some, z.amax(1, keepdim=True), 0.0)
    m = torch.where(torch.isneginf(m), 0.0, m)
    z = torch.where(ok, z - m, -math.inf)                                             # first: ln s would be lost beside 1e38
    s = torch.where(ok, z.exp(), 0.0).sum(1, keepdim=True)
    logp = torch.where(ok, z - torch.log(s), -math.inf)
    p = torch.where(ok, logp.exp(), 0.0)
    H = -torch.where(p > 0, p * logp, 0.0).sum(1)
    v = x.shape[1]
    a = actions
    lp = logp.gather(1, a.clamp(0, v - 1))
    lp = torch.where(a < 0, 0.0, lp)
    order = torch.sort(torch.where(ok, x, -math.inf), dim=1, descending=True, stable=True)
    k = min(top, v)
    ta, tl = order.indices[:, :k], logp.gather(1, order.indices[:, :k])
    ta = torch.where(torch.isneginf(order.values[:, :k]), -1, ta)
    ta = torch.nn.functional.pad(ta, (0, top - k), value=-1)
    tl = torch.nn.functional.pad(tl, (0, top - k), value=-math.inf)
    return lp, H, ta, tl, p, logp, ok


def gradient(ref, actions, g, h, temperature):
    """(dL/dx, the sum of its parts' sizes) in float64."""
    _, H, _, _, p, logp, ok = ref
    a = actions
    g = torch.where(a >= 0, g.double(), 0.0)
    d = torch.zeros_like(p).scatter_add_(1, a.clamp(min=0), g)
    G = g.sum(1, keepdim=True)
    h = h.double()[:, None]
    lp = torch.where(p > 0, logp, 0.0)
    dx = torch.where(ok, (d - p * G - h * p * (lp + H[:, None])) / temperature, 0.0)
    size = (torch.zeros_like(p).scatter_add_(1, a.clamp(min=0), g.abs()) + p * g.abs().sum(1, keepdim=True) + h.abs() * p * (lp.abs() + H[:, None])) / temperature
    return dx, size


def near(got, want, tol, what):
    got = got.double()
    want = torch.where(want < -torch.finfo(torch.float32).max, -math.inf, want)       # what float32 cannot hold
    assert torch.equal(torch.isfinite(got), torch.isfinite(want)), what + ": other places are finite"
    assert torch.equal(got[~torch.isfinite(want)], want[~torch.isfinite(want)]), what
    fin = torch.isfinite(want)
    over = ((got - want).abs() - tol)[fin]
    assert over.numel() == 0 or float(over.max()) <= 0, "%s: %.3g over its tolerance" % (what, float(over.max()))


def check(x, allowed, mask, actions, top=0, temperature=1.0, grads=True, seed=0):
    """One call against the definition: x [n, v], allowed bool [n, v], actions [n, k]."""
    from checkers_mcts_amd import policy
    n, v = x.shape
    leaf = x.detach().requires_grad_(grads)
    out = policy.action_logprobs(leaf, actions, mask=mask, top=top, temperature=temperature)
    ref = reference(x.detach(), allowed, actions.long(), top, temperature)
    b = bound(v)
    tol = lambda want: b + 4 * U * torch.where(torch.isfinite(want), want, 0.0).abs() + 4 * U * math.log(v + 1)
    near(out.logp.detach(), ref[0], tol(ref[0]), "logp")
    near(out.entropy.detach(), ref[1], b * (1 + 2 * (ref[1] + math.log(v))), "entropy")
    if top:
        assert torch.equal(out.top_action, ref[2]), "alternatives"
        near(out.top_logp, ref[3], tol(ref[3]), "top_logp")
        assert out.top_action.dtype == torch.int64
    if grads:
        gen = torch.Generator(device="cuda").manual_seed(seed + 77)
        g = torch.randn(actions.shape, generator=gen, device="cuda")
        h = torch.randn((n,), generator=gen, device="cuda")
        dx, = torch.autograd.grad((out.logp, out.entropy), (leaf,), (g, h))
        want, size = gradient(ref, actions.long(), g, h, temperature)
        # p carries B and 2 |log p| u, each product and sum one u more; then one rounding to the type, or half its smallest step
        t = size * (2 * b + 16 * U) + 4 * U * (ref[5].abs().nan_to_num(posinf=0.0) * size) + want.abs() * torch.finfo(x.dtype).eps / 2 + torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
        assert dx.dtype == x.dtype and dx.shape == x.shape
        near(dx, want, t, "gradient")
    return out


def make(n, v, dtype, seed, k=1, scale=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn((n, v), generator=g, device="cuda") * scale).to(dtype)
    a = torch.randint(-1, v, (n, k), generator=g, device="cuda")
    allowed = torch.rand((n, v), generator=g, device="cuda") < 0.7
    return x, a, allowed


SIZES = [(1, 1), (3, 2), (5, 7), (4, 63), (2, 64), (9, 65), (70, 128), (3, 511), (130, 512), (5, 513), (2, 1000), (7, 2047), (3, 2049), (5, 4097), (2, 8191),
         (1, 20000), (3, 50001), (1, 131072)]


@pytest.mark.parametrize("n,v", SIZES)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_sizes(n, v, dtype):
    x, a, allowed = make(n, v, dtype, n * 1000 + v, k=3)
    every = torch.ones_like(allowed)
    check(x, every, None, a, top=min(6, v), seed=v)
    check(x, allowed, allowed, a, top=9, temperature=0.7, seed=v + 1)


@pytest.mark.parametrize("n", [1, 2, 63, 300, 5000])
def test_legal_words_of_real_positions(n):
    from checkers_mcts_amd import rules, policy
    from test_rules_gpu import random_boards
    boards = rules.boards_to_device(random_boards(n, n))
    words, _ = rules.movegen(boards)
    allowed = policy.legal_from_features(rules.features(boards))
    if n <= 300:
        assert torch.equal(allowed, dark(words))
    x, a, _ = make(n, 512, torch.float32, n, k=4)
    one = check(x, allowed, words, a, top=12, temperature=1.3)
    two = policy.action_logprobs(x, a, mask=allowed, top=12, temperature=1.3)
    assert torch.equal(one.top_action, two.top_action)
    near(one.logp.detach(), two.logp.double(), 2 * bound(512) + 8 * U * two.logp.double().abs().nan_to_num(posinf=0.0), "words and bool")


def test_words_that_leave_no_action_and_all_of_them():
    words = torch.zeros((6, 8), dtype=torch.int32, device="cuda")
    words[1] = -1
    words[2, 3] = 1 << 30
    words[3, 7] = -(1 << 31)
    words[4, 0] = 0x0F0F0F0F
    x, _, _ = make(6, 512, torch.float32, 3)
    a = torch.randint(0, 512, (6, 5), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    out = check(x, dark(words), words, a, top=20)
    assert out.entropy[0] == 0 and torch.isneginf(out.logp[0]).all() and (out.top_action[0] == -1).all()
    assert out.top_logp[2, 0] == 0 and out.entropy[2] == 0
    check(x, dark(words[4:5]).expand(6, 512), words[4], a, top=20)                    # one mask for every row


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("v", [5, 512, 3000, 40000])
def test_rows_without_an_allowed_action(dtype, v):
    x, a, allowed = make(5, v, dtype, v, k=2)
    a = a.clamp(min=0)
    a[4] = -1
    allowed[1] = False
    x[2] = -math.inf                                                                  # masked by the logits themselves
    allowed[4] = False
    out = check(x, allowed, allowed, a, top=4)
    for r in (1, 2):
        assert torch.isneginf(out.logp[r]).all() and out.entropy[r] == 0 and (out.top_action[r] == -1).all() and torch.isneginf(out.top_logp[r]).all()
    assert (out.logp[4] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("v", [3, 512, 5000, 33000])
def test_lowest_and_largest_values(dtype, v):
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    x, a, allowed = make(6, v, dtype, v + 9, k=2)
    x[0] = low                                                                        # all of it: uniform
    x[1] = torch.where(allowed[1], x[1], low)
    x[2] = high
    x[3, ::2] = low
    x[3, v // 2] = high
    x[4] = -math.inf
    x[4, v - 1] = low                                                                 # the only one left
    x[5] = torch.where(allowed[5], low, -math.inf)
    a = a.clamp(min=0)
    a[3] = v // 2
    a[4] = v - 1
    a[1] = allowed[1].float().argmax()
    out = check(x, torch.ones_like(allowed), None, a, top=3)
    assert abs(float(out.entropy[0]) - math.log(v)) <= bound(v) * (1 + 4 * math.log(v + 1))
    assert out.top_action[4].tolist() == [v - 1, -1, -1] and float(out.logp[4, 0]) == 0


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("v", [9, 512, 5000, 70000])
def test_what_is_masked_may_hold_anything(dtype, v):
    x, a, allowed = make(4, v, dtype, v + 3, k=2)
    allowed[:, 0] = True
    allowed[2] = False
    a = torch.where(allowed.gather(1, a.clamp(min=0)), a, torch.zeros_like(a))
    clean = check(x, allowed, allowed, a, top=5)
    dirty = x.clone()
    junk = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(dtype).max, torch.finfo(dtype).min], device="cuda").to(dtype)
    junk = junk[torch.arange(v, device="cuda") % 5].expand(4, v)
    dirty = torch.where(allowed, x, junk)
    from checkers_mcts_amd import policy
    leaf = dirty.requires_grad_(True)
    out = policy.action_logprobs(leaf, a, mask=allowed, top=5)
    for got, want in zip(out, clean):
        assert torch.equal(got, want)
    g1, = torch.autograd.grad((out.logp.nan_to_num(neginf=0.0).sum() + out.entropy.sum()), leaf)
    assert torch.isfinite(g1).all() and (g1[~allowed] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("v", [6, 512, 5000, 70000])
def test_nan_and_infinity_among_the_allowed(dtype, v):
    from checkers_mcts_amd import policy
    x, a, allowed = make(4, v, dtype, v + 5)
    a = a.clamp(min=0)
    x[0, v // 2] = math.nan
    x[1, v - 1] = math.inf
    x[3, 0] = math.nan
    mask = torch.ones_like(allowed)
    mask[3, 0] = False
    leaf = x.requires_grad_(True)
    out = policy.action_logprobs(leaf, a, mask=mask, top=3)
    for r in (0, 1):
        assert out.logp[r].isnan().all() and out.entropy[r].isnan() and out.top_logp[r].isnan().all() and (out.top_action[r] == -1).all()
    assert torch.isfinite(out.entropy[2:]).all() and (out.top_action[2:] >= 0).all()
    g, = torch.autograd.grad(out.entropy.sum(), leaf)
    assert g[0].isnan().all() and g[1].isnan().all() and torch.isfinite(g[2:]).all()
    a = torch.full_like(a, -1)
    assert (policy.action_logprobs(x.detach(), a, mask=mask).logp == 0).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("v", [40, 512, 4000, 66000])
def test_ties_go_to_the_lowest_action(dtype, v):
    from checkers_mcts_amd import policy
    g = torch.Generator(device="cuda").manual_seed(v)
    x = torch.randint(-2, 3, (5, v), generator=g, device="cuda").to(dtype)
    x[0] = 1.0
    x[1] = -0.0
    x[1, 1::2] = 0.0
    x[2] = torch.where(torch.arange(v, device="cuda") >= v - 3, 9.0, 0.0)
    out = check(x, torch.ones(5, v, dtype=torch.bool, device="cuda"), None, torch.zeros((5, 1), dtype=torch.long, device="cuda"), top=30)
    assert out.top_action[0].tolist() == list(range(30)) and out.top_action[1].tolist() == list(range(30))
    assert out.top_action[2, :3].tolist() == [v - 3, v - 2, v - 1]
    rising = torch.arange(v, device="cuda").to(torch.float32)[None].repeat(2, 1)
    rising[1] = rising[1].flip(0)
    out = policy.action_logprobs(rising, top=64 if v > 64 else v)
    k = out.top_action.shape[1]
    assert out.top_action.tolist() == [list(range(v - 1, v - 1 - k, -1)), list(range(k))]


def test_sixty_four_given_actions_and_alternatives_and_the_same_one_twice():
    for v in (5, 64, 512, 9001):
        x, a, allowed = make(3, v, torch.float32, v, k=64)
        a[:, 1] = a[:, 0] = 2
        a[1] = 4
        check(x, torch.ones_like(allowed), None, a, top=64)
        check(x, allowed, allowed, a, top=64)


def test_given_actions_beyond_the_row():
    from checkers_mcts_amd import policy
    x, a, _ = make(4, 700, torch.bfloat16, 1)
    a = a.clamp(min=0)
    a[1], a[2] = 700, 1 << 40
    leaf = x.requires_grad_(True)
    out = policy.action_logprobs(leaf, a[:, 0], top=2)
    assert out.logp.isnan().tolist() == [False, True, True, False] and torch.isfinite(out.entropy).all()
    g, = torch.autograd.grad(out.logp.sum(), leaf)
    assert g.isnan().all(1).tolist() == [False, True, True, False]
    a32 = torch.tensor([5, 699, -1, -2 ** 31], dtype=torch.int32, device="cuda")
    b = policy.action_logprobs(x.detach(), a32).logp
    assert torch.equal(b, policy.action_logprobs(x.detach(), a32.long()).logp) and b[2] == 0 and b[3] == 0


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("start", [0, 1, 3, 8])
@pytest.mark.parametrize("stride", [777, 778, 1024])
def test_rows_that_start_anywhere(dtype, start, stride):
    from checkers_mcts_amd import policy
    v, n = 777, 9
    buf = torch.full((n * stride + 16,), math.nan, device="cuda", dtype=dtype)
    x = buf.as_strided((n, v), (stride, 1), start)
    y, a, allowed = make(n, v, dtype, start + stride, k=2)
    x.copy_(y)
    check(x, torch.ones_like(allowed), None, a, top=5)
    big = torch.zeros((n, v + start + 2), dtype=torch.bool, device="cuda")
    mask = big[:, start:start + v]
    mask.copy_(allowed)
    check(x, allowed, mask, a, top=5)
    outside = torch.ones_like(buf, dtype=torch.bool).as_strided((n, v), (stride, 1), start)
    assert outside.all()


def test_other_orders_broadcasts_and_dimensions():
    from checkers_mcts_amd import policy
    y, a, allowed = make(600, 6, torch.float32, 4)
    x = y.t()                                                                         # [6, 600], the last dimension not dense
    a = torch.randint(0, 600, (6, 2), device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    leaf = y.clone().requires_grad_(True)
    out = policy.action_logprobs(leaf.t(), a, top=3)
    want = policy.action_logprobs(x.contiguous(), a, top=3)
    assert all(torch.equal(p, q) for p, q in zip(out, want))
    g, = torch.autograd.grad(out.logp.sum(), leaf)
    z = x.contiguous().requires_grad_(True)
    h, = torch.autograd.grad(policy.action_logprobs(z, a).logp.sum(), z)
    assert torch.equal(g, h.t())
    # one row for everybody: its gradient is the sum
    row = torch.randn((900,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).requires_grad_(True)
    acts = torch.arange(50, device="cuda")
    out = policy.action_logprobs(row.expand(50, 900), acts)
    g, = torch.autograd.grad(out.logp.sum(), row)
    p = torch.softmax(row.detach().double(), 0)
    want = (torch.arange(900, device="cuda") < 50).double() - 50 * p
    assert float((g.double() - want).abs().max()) <= 50 * bound(900) + 60 * U
    one = policy.action_logprobs(row.detach(), torch.tensor(7, device="cuda"), top=2)   # a single row, no leading dimension
    assert one.logp.shape == () and one.entropy.shape == () and one.top_action.shape == (2,)
    many = policy.action_logprobs(row.detach(), torch.tensor([7, 8], device="cuda"))
    assert many.logp.shape == (2,) and many.logp[0] == one.logp
    cube = torch.randn((3, 4, 100), device="cuda", generator=torch.Generator(device="cuda").manual_seed(5))
    acts = torch.randint(0, 100, (3, 4), device="cuda", generator=torch.Generator(device="cuda").manual_seed(5))
    keep = torch.rand((4, 100), device="cuda", generator=torch.Generator(device="cuda").manual_seed(6)) < 0.5
    out = policy.action_logprobs(cube, acts, mask=keep, top=2)
    flat = policy.action_logprobs(cube.reshape(12, 100), acts.reshape(12), mask=keep.repeat(3, 1), top=2)
    assert out.logp.shape == (3, 4) and out.entropy.shape == (3, 4) and out.top_logp.shape == (3, 4, 2)
    assert torch.equal(out.logp.reshape(12), flat.logp) and torch.equal(out.top_action.reshape(12, 2), flat.top_action)
    view = cube.transpose(0, 1)
    assert torch.equal(policy.action_logprobs(view, acts.t()).logp, policy.action_logprobs(cube, acts).logp.t())


def test_no_rows():
    from checkers_mcts_amd import policy
    out = policy.action_logprobs(torch.zeros((0, 50), device="cuda", requires_grad=True), torch.zeros((0, 2), dtype=torch.long, device="cuda"), top=3)
    assert out.logp.shape == (0, 2) and out.entropy.shape == (0,) and out.top_action.shape == (0, 3)
    out.entropy.sum().backward()


@pytest.mark.parametrize("v", [512, 1500, 30000])
def test_gradient_against_differences(v):
    from checkers_mcts_amd import policy
    x, a, allowed = make(4, v, torch.float32, v + 1, k=2)
    allowed[:, :3] = True
    a = torch.randint(0, 3, (4, 2), device="cuda", generator=torch.Generator(device="cuda").manual_seed(8))
    leaf = x.clone().requires_grad_(True)
    out = policy.action_logprobs(leaf, a, mask=allowed, temperature=0.9)
    w = torch.tensor([[0.3, -1.0], [2.0, 0.1], [0.0, 1.0], [-0.5, -0.5]], device="cuda")
    g, = torch.autograd.grad((out.logp * w).sum() - 0.7 * out.entropy.sum(), leaf)

    def loss(y):
        lp, H = reference(y, allowed, a, 1, 0.9)[:2]
        return float((lp * w.double()).sum() - 0.7 * H.sum())
    for s in range(6):
        u = torch.randn(x.shape, generator=torch.Generator(device="cuda").manual_seed(s), device="cuda", dtype=torch.float64)
        if s < 3:
            u = torch.zeros_like(u).index_fill_(1, torch.tensor([s], device="cuda"), 1.0)
        e = 1e-4
        diff = (loss(x.double() + e * u) - loss(x.double() - e * u)) / (2 * e)
        got = float((g.double() * u).sum())
        # the third derivative's e^2 / 6 and the differences' own rounding; then the kernel's
        assert abs(got - diff) <= 1e-6 * (1 + abs(diff)) + bound(v) * 30 * float((g.double().abs() * u.abs()).sum())


def test_saved_tensors_that_come_back_elsewhere_and_two_backward_passes():
    from checkers_mcts_amd import policy
    x, a, allowed = make(40, 3000, torch.float32, 6, k=2)
    a = a.clamp(min=0)
    want = None
    for hooks in (False, True):
        leaf = x.clone().requires_grad_(True)
        if hooks:
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.cuda()):
                out = policy.action_logprobs(leaf, a, mask=allowed, top=3)
        else:
            out = policy.action_logprobs(leaf, a, mask=allowed, top=3)
        g = torch.ones_like(out.logp.detach())
        one, = torch.autograd.grad((out.logp, out.entropy), leaf, (g, torch.ones(40, device="cuda")), retain_graph=True)
        two, = torch.autograd.grad(out.entropy.sum(), leaf, retain_graph=True)         # without the given actions, then with them again
        three, = torch.autograd.grad((out.logp, out.entropy), leaf, (g, torch.ones(40, device="cuda")))
        assert torch.equal(one, three) and not torch.equal(one, two)
        want = want or (one, two)
        assert torch.equal(one, want[0]) and torch.equal(two, want[1])
    leaf = x.clone().requires_grad_(True)
    out = policy.action_logprobs(leaf * 1.0, a, mask=allowed)
    allowed.logical_not_()
    with pytest.raises(RuntimeError, match="inplace"):
        out.entropy.sum().backward()


def test_large_offsets():
    from checkers_mcts_amd import policy
    n, v = 66000, 32768                                                               # 2.16e9 logits: offsets beyond 32 bits
    x = torch.zeros((n, v), dtype=torch.float16, device="cuda")
    rows = torch.tensor([0, 1, 65535, 65536, n - 1], device="cuda")
    x[rows] = torch.randn((5, v), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").half()
    a = torch.full((n,), v - 1, device="cuda")
    out = policy.action_logprobs(x.requires_grad_(True), a, top=3)
    ref = reference(x.detach()[rows], torch.ones((5, v), dtype=torch.bool, device="cuda"), a[rows][:, None], 3, 1.0)
    near(out.logp.detach()[rows], ref[0][:, 0], 2 * bound(v) + 8 * U * ref[0][:, 0].abs(), "logp")
    assert torch.equal(out.top_action[rows], ref[2])
    other = torch.ones((n,), dtype=torch.bool, device="cuda")
    other[rows] = False
    assert float((out.entropy.detach()[other].double() - math.log(v)).abs().max()) <= bound(v) * 30
    g, = torch.autograd.grad(out.entropy.sum() + out.logp.sum(), x)
    del x, out
    want, size = gradient(ref, a[rows][:, None], torch.ones((5, 1), device="cuda"), torch.ones((5,), device="cuda"), 1.0)
    near(g[rows], want, size * (4 * bound(v) + 64 * U) + want.abs() * 2.0 ** -11 + 2.0 ** -25, "gradient")


@pytest.mark.parametrize("n,v", [((1 << 25) + 9, 3), ((1 << 23) + 5, 16384 + 1)])
def test_more_rows_than_a_launch_takes(n, v):
    from checkers_mcts_amd import policy
    row = torch.randn((v,), generator=torch.Generator(device="cuda").manual_seed(4), device="cuda").half()
    a = torch.full((n,), 1, dtype=torch.int32, device="cuda")
    out = policy.action_logprobs(row.expand(n, v), a, top=1)
    one = reference(row[None], torch.ones((1, v), dtype=torch.bool, device="cuda"), torch.ones((1, 1), dtype=torch.long, device="cuda"), 1, 1.0)
    assert bool((out.logp == out.logp[0]).all()) and bool((out.entropy == out.entropy[0]).all()) and bool((out.top_action == one[2][0, 0]).all())
    near(out.logp[:1], one[0][0], bound(v) + 4 * U * one[0][0].abs() + 64 * U, "logp")
    near(out.entropy[-1:], one[1], bound(v) * (1 + 2 * (one[1] + math.log(v))), "entropy")


@pytest.mark.parametrize("n", [1, 3, 700, 1100, 2047, 2048, 2500])
@pytest.mark.parametrize("v", [2049, 8193, 16384, 16500])
def test_rows_shared_by_a_workgroup(n, v):
    """Around the sizes at which a row goes from a wavefront to a workgroup and to several."""
    x, a, allowed = make(n, v, torch.bfloat16, n + v, k=2)
    check(x, allowed, allowed, a, top=7, grads=n < 1000, seed=v)
    y = (x.float() / 8).round()                                                       # many ties
    check(y, torch.ones_like(allowed), None, a, top=20, grads=False)


@pytest.mark.parametrize("n,v,dtype,masked", [(2557, 16411, torch.float32, True), (2555, 16411, torch.float32, False), (2600, 32771, torch.bfloat16, False)], ids=str)
def test_gradients_on_both_sides_of_the_caches(n, v, dtype, masked):
    """Around 160 MiB, from which on they are stored past the caches."""
    x, a, allowed = make(n, v, dtype, n, k=2)
    check(x, allowed if masked else torch.ones_like(allowed), allowed if masked else None, a, seed=n)


def test_another_stream_and_two_calls_at_once():
    from checkers_mcts_amd import policy
    x, a, allowed = make(64, 20000, torch.float32, 2, k=2)
    y, b, keep = make(3, 90000, torch.bfloat16, 3, k=1)
    want = policy.action_logprobs(x, a, mask=allowed, top=8), policy.action_logprobs(y, b, mask=keep, top=8)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(5):
        with torch.cuda.stream(s1):
            p = policy.action_logprobs(x, a, mask=allowed, top=8)
        with torch.cuda.stream(s2):
            q = policy.action_logprobs(y, b, mask=keep, top=8)
        got.append((p, q))
    torch.cuda.synchronize()
    for p, q in got:
        assert all(torch.equal(i, j) for i, j in zip(p, want[0])) and all(torch.equal(i, j) for i, j in zip(q, want[1]))


@pytest.mark.parametrize("n,v", [(1, 512), (40, 3000), (2, 100000)])
def test_captured_forward_and_backward(n, v):
    from checkers_mcts_amd import policy
    x, a, allowed = make(n, v, torch.bfloat16, v, k=2)
    g = torch.ones((n, 2), device="cuda")
    h = torch.ones((n,), device="cuda")

    def both(x):
        leaf = x.detach().requires_grad_(True)
        out = policy.action_logprobs(leaf, a, mask=allowed, top=4, temperature=0.8)
        return [t.detach() for t in out] + list(torch.autograd.grad((out.logp, out.entropy), (leaf,), (g, h)))
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        both(x)
    torch.cuda.current_stream().wait_stream(warm)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):                                                                # two graphs, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = both(x)
        graphs.append((graph, outs))
    for rep in range(4):
        x.copy_(make(n, v, torch.bfloat16, v + rep, k=2)[0])
        want = both(x)
        for graph, outs in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, outs in graphs:
            assert all(torch.equal(p, q) for p, q in zip(outs, want))


def test_rank_moves_agrees_with_the_masked_softmax():
    from checkers_mcts_amd import policy, rules, net as N
    from test_rules_gpu import random_boards
    boards = rules.boards_to_device(random_boards(200, 5))
    net = N.make_net(128, seed=3)
    x = rules.features(boards)
    z, value = net.logits(x.permute(0, 3, 1, 2))
    p, value2 = net(x.permute(0, 3, 1, 2))
    assert float((torch.softmax(z, 1) - p).abs().max()) <= 1e-5 and float((value - value2).abs().max()) <= 1e-5

    class Same:                                                                       # the same logits for both: library convolutions need not repeat bit for bit
        parameters, logits = net.parameters, lambda self, x: (z, value)
    got = policy.rank_moves(net, boards, top=6)
    assert got.action.shape == (200, 6) and float((got.value - value).abs().max()) <= 1e-5
    got = policy.rank_moves(Same(), boards, top=6)
    dense = rules.mask_renorm(boards, torch.softmax(z, 1).contiguous())
    legal = policy.legal_from_features(x)
    for i in range(200):
        k = min(6, int(legal[i].sum()))
        assert (got.action[i, k:] == -1).all()
        mine = got.action[i, :k]
        assert legal[i][mine].all()
        # both are float32 softmaxes over the same logits: 512-term sums in other orders
        assert float((got.logp[i, :k].exp() - dense[i][mine]).abs().max() if k else 0.0) <= 64 * U
        assert k == 0 or float(dense[i].max() - dense[i][mine[0]]) <= 64 * U


def test_entropy_weight_and_policy_figures_of_training():
    from checkers_mcts_amd import policy, rules, train, net as N
    from test_train_hip_gpu import make_batch
    x, pi, tv = make_batch(64, 4)
    net = train.create_nn(NUM_KERNELS=32, CONV_REG=1e-3, DENSE_REG=1e-3, POLICY_LOSS_WEIGHT=1.0, VALUE_LOSS_WEIGHT=1.0, SEED=2).cuda()
    net.eval()
    base, ce, mse = train.losses(net, x, pi, tv, with_penalty=False)
    with_entropy, _, _ = train.losses(net, x, pi, tv, with_penalty=False, entropy_weight=0.25)
    z, _ = net.logits(x.permute(0, 3, 1, 2))
    legal = policy.legal_from_features(x)
    ref = reference(z.detach(), legal, pi.argmax(1)[:, None], 3, 1.0)
    assert abs(float(base - with_entropy) - 0.25 * float(ref[1].mean())) <= 1e-5
    g1 = torch.autograd.grad(with_entropy, net.pol_fc.bias)[0]
    g0 = torch.autograd.grad(base, net.pol_fc.bias)[0]
    want, _ = gradient(ref, pi.argmax(1)[:, None], torch.zeros((64, 1), device="cuda"), torch.full((64,), -0.25 / 64, device="cuda"), 1.0)
    assert float((g1.double() - g0.double() - want.sum(0)).abs().max()) <= 1e-6
    figures = train.policy_figures(net, x, pi)
    assert abs(float(figures[0] - ref[1].sum())) <= 64 * bound(512) * 20
    hits = (ref[2] == pi.argmax(1)[:, None]).any(1).sum()
    assert float(figures[2]) == float(hits)


def test_policy_figures_of_positions_without_visits():
    """Games that run to their end leave terminal tuples: no visits, no legal move.  The figures are those of the other rows."""
    from checkers_mcts_amd import engine as E, policy, train
    from test_engine_gpu import mk, run_engine
    eng, ev = run_engine(E, mk(6), [3, 4, 5], games_per_slot=2, terminate_cnt=400)
    eng.run(ev)
    data = train.TrainingData(tuples=eng.pack_tuples_device())
    x, pi, tv = data.batch(torch.arange(len(data), device="cuda"))
    eng.close()
    played = pi.sum(1) > 0
    assert 0 < int((~played).sum()) < 64 and not policy.legal_from_features(x)[~played].any()
    net = train.create_nn(NUM_KERNELS=32, CONV_REG=1e-3, DENSE_REG=1e-3, POLICY_LOSS_WEIGHT=1.0, VALUE_LOSS_WEIGHT=1.0, SEED=2).cuda().eval()
    sel = torch.cat([torch.nonzero(~played)[:, 0], torch.nonzero(played)[:200, 0]])
    x, pi, tv, played = x[sel], pi[sel], tv[sel], played[sel]
    with torch.no_grad():
        z, _ = net.logits(x[played].permute(0, 3, 1, 2))
    move = pi[played].argmax(1)
    ref = reference(z, policy.legal_from_features(x[played]), move[:, None], 3, 1.0)
    n = int(played.sum())
    figures = train.policy_figures(net, x, pi).tolist()
    assert figures[3] == n
    # a library convolution over another batch may sum in another order: 1e-5 of a logit, as the network's own tests have it
    assert abs(figures[0] - float(ref[1].sum())) <= n * (20 * bound(512) + 1e-4) and abs(figures[1] - float(ref[0].sum())) <= n * (2 * bound(512) + 1e-4)
    assert abs(figures[2] - float((ref[2] == move[:, None]).any(1).sum())) <= 2          # two nearly equal candidates may change places
    none = train.policy_figures(net, x[~played], pi[~played]).tolist()
    assert none == [0.0, 0.0, 0.0, 0.0]
    with torch.autocast("cuda", dtype=torch.bfloat16), torch.no_grad():
        z16, _ = net.logits(x[played].permute(0, 3, 1, 2))
    ref = reference(z16, policy.legal_from_features(x[played]), move[:, None], 3, 1.0)
    half = train.policy_figures(net, x, pi, torch.bfloat16).tolist()                     # as the losses beside them are computed
    # bfloat16 logits of size |z|: a last bit up or down is 2^-7 |z|, in the row's sum too
    assert abs(half[1] - float(ref[0].sum())) <= n * (2 * bound(512) + 2 * 2.0 ** -7 * float(z16.abs().max()))


def test_train_nn_policy_metrics_of_whole_games(tmp_path, monkeypatch):
    import numpy as np
    from checkers_mcts_amd import engine as E, train
    from test_engine_gpu import mk, run_engine
    monkeypatch.chdir(tmp_path)
    eng, ev = run_engine(E, mk(6), [3, 4, 5], games_per_slot=2, terminate_cnt=400)
    eng.run(ev)
    tuples = eng.pack_tuples_device()
    eng.close()
    data = train.TrainingData(tuples=tuples)
    _, pi, _ = data.batch(torch.arange(len(data), device="cuda"))
    last = torch.nonzero(pi.sum(1) == 0)[:, 0]
    assert len(last)
    kw = dict(PATIENCE=5, MIN_DELTA=0, VAL_SPLIT=0.5, TRAINING_ITERATION=0, BATCH_SIZE=32, CLR_SS_COEFF=4, NN_BASE_LR=1e-4, NN_MAX_LR=1e-3, EPOCHS=2, NUM_KERNELS=32,
              CONV_REG=1e-4, DENSE_REG=1e-4, POLICY_LOSS_WEIGHT=1.0, VALUE_LOSS_WEIGHT=1.0, SEED=1, TRAIN_BACKEND="torch", POLICY_METRICS=True)
    # every second row of the job is one of a game's end
    many = torch.cat([tuples[:200], tuples[last].repeat(200 // len(last) + 1, 1)])
    history, _ = train.train_nn(many.contiguous(), train.create_nn(**kw), **kw)
    h = history.history
    assert all(np.isfinite(h[k]).all() for k in ("val_policy_entropy", "val_move_logp", "val_move_top3"))
    assert max(h["val_move_logp"]) < 0 and min(h["val_policy_entropy"]) > 0 and 0 <= min(h["val_move_top3"]) <= 1
    only = tuples[last].repeat(200 // len(last) + 1, 1).contiguous()                     # nothing to speak of
    h = train.train_nn(only, train.create_nn(**kw), **kw)[0].history
    assert all(np.isnan(h[k]).all() for k in ("val_policy_entropy", "val_move_logp", "val_move_top3"))


def test_gradients_that_are_seen_negated():
    """The gradient of an imaginary part may come as a view of its conjugate: the memory holds the opposite sign."""
    from checkers_mcts_amd import policy
    x, a, _ = make(1, 700, torch.float32, 5)
    a = a.clamp(min=0)[:, 0]
    for name in ("logp", "entropy"):
        leaf = x.clone().requires_grad_(True)
        out = getattr(policy.action_logprobs(leaf, a), name)
        one = torch.ones_like(out)
        want, = torch.autograd.grad(out, leaf, -one, retain_graph=True)
        seen = []
        out.register_hook(lambda g: seen.append(g.is_neg()))
        got, = torch.autograd.grad((torch.complex(one, out).conj() * torch.complex(one, 3 * one)).imag.sum(), leaf)      # 3 - out
        assert seen == [True] and torch.equal(got, want)


def test_derivatives_that_are_not_there_are_refused():
    """Forward-mode derivatives and recorded programs: neither would see what the kernels do."""
    import torch.autograd.forward_ad as forward_ad
    from checkers_mcts_amd import policy
    x, a, _ = make(4, 20, torch.float32, 1)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for leaf in (dual, dual.reshape(2, 2, 20)):
            with pytest.raises((ValueError, NotImplementedError)):
                policy.action_logprobs(leaf)
        with torch.no_grad(), pytest.raises((ValueError, NotImplementedError)):
            policy.action_logprobs(dual, a)
        inside = policy.action_logprobs(x, a)                          # without a tangent: as ever
    assert all(torch.equal(p, q) for p, q in zip(inside[:2], policy.action_logprobs(x, a)[:2]))
    entropy = lambda t: policy.action_logprobs(t).entropy
    with pytest.raises((ValueError, RuntimeError)):
        torch.func.jvp(entropy, (x,), (torch.ones_like(x),))
    with pytest.raises((ValueError, RuntimeError)):
        torch.func.vmap(entropy)(x[None])
    with pytest.raises(ValueError, match="record"):
        torch.jit.trace(entropy, (x,), check_trace=False)
    from torch.fx.experimental.proxy_tensor import make_fx
    with pytest.raises(ValueError, match="record"):
        make_fx(entropy)(x)
    assert torch.equal(entropy(x), policy.action_logprobs(x, a).entropy)


@pytest.mark.parametrize("temperature", [4.0, 1e3, 1e6])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("v", [5, 512, 5000])
def test_differences_beyond_float32_are_scaled_first(dtype, v, temperature):
    """x - max may not fit where (x - max) / temperature does: lowest against largest values."""
    x, a, allowed = make(6, v, dtype, v, k=3)
    far = torch.finfo(dtype).max
    x[:, 0], x[:, v - 1], x[:, 2] = far, -far, far * 0.75
    a[:, 0], a[:, 1] = v - 1, 0
    x[3] = -far
    check(x, torch.ones_like(allowed), None, a, top=5, temperature=temperature, grads=False)


def test_losses_of_16_bit_logits_with_an_entropy_term():
    """The softmax of the loss is float32 with the term as without it."""
    from checkers_mcts_amd import train
    from test_train_hip_gpu import make_batch
    x, pi, tv = make_batch(64, 4)
    z = (torch.randn((64, 512), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda") * 3).bfloat16()

    class Net:
        policy_loss_weight = value_loss_weight = 1.0

        def logits(self, x):
            return z, tv * 0.5

        def __call__(self, x):
            return torch.softmax(z.float(), 1), tv * 0.5
    without = train.losses(Net(), x, pi, tv, with_penalty=False)
    with_term = train.losses(Net(), x, pi, tv, with_penalty=False, entropy_weight=0.25)
    assert torch.equal(without[1], with_term[1]) and torch.equal(without[2], with_term[2])


def test_leaving_the_hand_written_training_step_is_said(tmp_path, monkeypatch):
    import warnings
    from checkers_mcts_amd import train
    from test_train_hip_gpu import make_batch
    monkeypatch.chdir(tmp_path)
    data = train.TrainingData(dense=make_batch(64, 6))
    kw = dict(PATIENCE=5, MIN_DELTA=0, VAL_SPLIT=0.0, TRAINING_ITERATION=0, BATCH_SIZE=32, CLR_SS_COEFF=4, NN_BASE_LR=1e-4, NN_MAX_LR=1e-3, EPOCHS=1, NUM_KERNELS=128,
              CONV_REG=1e-4, DENSE_REG=1e-4, POLICY_LOSS_WEIGHT=1.0, VALUE_LOSS_WEIGHT=1.0, SEED=1, MODEL_SUFFIX=".pt")
    for more, said in ((dict(OPTIMIZER="adamw"), True), (dict(ENTROPY_WEIGHT=0.01), True), (dict(), False), (dict(OPTIMIZER="adamw8", TRAIN_BACKEND="torch"), False)):
        with warnings.catch_warnings(record=True) as caught:
            warnings.simplefilter("always")
            train.train_nn(data, train.create_nn(**kw), **dict(kw, **more))
        said_now = [str(w.message) for w in caught if issubclass(w.category, RuntimeWarning) and "hand-written" in str(w.message)]
        assert bool(said_now) == said and all("OPTIMIZER" in m and "ENTROPY_WEIGHT" in m for m in said_now), (more, said_now)


def test_policy_figures_take_the_precision_around_them():
    from checkers_mcts_amd import train
    from test_train_hip_gpu import make_batch
    x, pi, _ = make_batch(8, 4)
    seen = []

    class Net:
        def logits(self, x):
            seen.append(torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled("cuda") else None)
            return torch.zeros((8, 512), device="cuda"), None
    train.policy_figures(Net(), x, pi)
    train.policy_figures(Net(), x, pi, torch.float32)
    train.policy_figures(Net(), x, pi, torch.bfloat16)
    with torch.autocast("cuda", dtype=torch.float16):
        train.policy_figures(Net(), x, pi)
    assert seen == [None, None, torch.bfloat16, torch.float16]
