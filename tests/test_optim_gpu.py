"""GPU: optim.AdamW (csrc/ckr_adamw.hip) against its formula in float64: three types, moments in 32 and 8 bits, clipping, odd and empty
tensors, more of them than one launch takes, missing gradients, layouts and alignments, captured steps, checkpoints; the 8-bit codes are
compared one by one, their rounding on average; and the operators together with policy.action_logprobs as a training step.

Tolerances (u = 2^-24): m = b1 m + a1 g and v = b2 v + a2 g^2 are 3 and 4 roundings of their parts; the update lr / bc1 * m / (sqrt(v) rs +
eps) adds a root, a product, a sum, a quotient, a product and the rounded factors: 12 u of its size, and what m's cancellation leaves of its parts'
size; w adds 2 u |w|.  A 16-bit parameter is the rounding of its master copy."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DTYPES = (torch.float32, torch.bfloat16, torch.float16)
SIZES = (1, 7, 8, 127, 128, 129, 2047, 2048, 2049, 5001, 70000)


# ---- the 8-bit formats from their definition, in float64 ---------------------------------------------------------------------------
def philox(seed, groups, step):
    """Philox4x32-10, key = seed, counter = (group, 0, step, 0): [groups, 4] words."""
    def mul(a, b):
        lo = (a & 0xFFFF) * b
        hi = (a >> 16) * b + (lo >> 16)
        return hi >> 16, ((hi & 0xFFFF) << 16) | (lo & 0xFFFF)
    i = groups.long()
    c0, c1, c2, c3 = i & 0xFFFFFFFF, i >> 32, torch.full_like(i, step), torch.zeros_like(i)
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(10):
        h0, l0 = mul(c0, 0xD2511F53)
        h1, l1 = mul(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return torch.stack((c0, c1, c2, c3), 1)


def dithers(seed, first, n, step):
    """16 dither bits of m and of v for elements first ... first + n - 1 of the states."""
    w = philox(seed, torch.arange(first // 8, (first + n) // 8, device="cuda"), step)
    lo, hi = (w & 0xFFFF), (w >> 16)
    return torch.stack((hi, lo), 2).reshape(-1), torch.stack((lo, hi), 2).reshape(-1)


def rounded(x, powers, dither, raise_small):
    """The value a code holds for x: 3 mantissa bits after adding (2 dither + 1) / 2^17 of a step to the first 20; `powers` powers of two below the scale."""
    fr, ex = torch.frexp(x.abs())
    eighths = torch.floor((torch.floor(fr * 2.0 ** 21) + (2 * dither + 1).double()) / 2.0 ** 17)
    y = torch.ldexp(eighths / 8, ex - 1)
    top = torch.frexp(x.abs().view(-1, 128).amax(1))[1].clamp(min=-126)
    least = torch.ldexp(torch.tensor(1.125, dtype=torch.float64, device=x.device), top + 1 - powers).repeat_interleave(128)
    y = torch.where(y < least, least if raise_small else torch.zeros_like(y), y)
    return torch.where(x == 0, 0.0, y * x.sign())


class Reference:
    """AdamW in float64, one tensor at a time; with bits = 8 the moments hold the codes' values."""

    def __init__(self, opt, lr, wd, betas, eps, bits, seed, max_norm=None):
        self.lr, self.wd, self.b, self.eps, self.bits, self.seed, self.max_norm = lr, wd, betas, eps, bits, seed, max_norm
        self.w = [p.detach().double().clone() for p in opt.params]
        self.m = [torch.zeros_like(w) for w in self.w]
        self.v = [torch.zeros_like(w) for w in self.w]
        self.t = [0] * len(self.w)
        self.off = opt.offsets

    def step(self, grads):
        b1, b2 = self.b
        c = 1.0
        if self.max_norm is not None:
            self.norm = math.sqrt(sum(float(g.double().square().sum()) for g in grads if g is not None))
            c = min(1.0, self.max_norm / (self.norm + 1e-6))
        self.size = []
        for i, g in enumerate(grads):
            if g is None:
                self.size.append(torch.zeros_like(self.w[i]))
                continue
            self.t[i] += 1
            t, g = self.t[i], g.double() * c
            ms = (b1 * self.m[i]).abs() + ((1 - b1) * g).abs()
            m, v = b1 * self.m[i] + (1 - b1) * g, b2 * self.v[i] + (1 - b2) * g * g
            rate, den = self.lr / (1 - b1 ** t), (v / (1 - b2 ** t)).sqrt() + self.eps
            self.w[i] = self.w[i] * (1 - self.lr * self.wd) - rate * m / den
            self.size.append(2 * self.w[i].abs() + rate * (12 * m.abs() + 3 * ms) / den)
            if self.bits == 8:
                n = m.numel()
                pad = (n + 127) // 128 * 128
                rm, rv = dithers(self.seed, self.off[i], pad, t)
                flat = lambda x: torch.nn.functional.pad(x.reshape(-1), (0, pad - n))
                m, v = rounded(flat(m), 16, rm, False)[:n].view_as(m), rounded(flat(v), 32, rv, True)[:n].view_as(v)
            self.m[i], self.v[i] = m, v


def make(sizes, dtype, seed, scale=0.1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn((n,), generator=g, device="cuda") * scale).to(dtype) for n in sizes]


def compare(opt, ref, drift):
    """drift: the steps so far (each adds its own roundings)."""
    m, v = opt.moments()
    if opt.master is not None:
        masters = opt.split(opt.master)
    for i, (p, w) in enumerate(zip(opt.params, ref.w)):
        got = (masters[i] if p.dtype != torch.float32 else p).detach().double()
        err = (got - w).abs() - ref_size[i] * U * 1.01
        assert p.numel() == 0 or float(err.max()) <= 0, "tensor %d: %.3g over its tolerance" % (i, float(err.max()))
        if p.dtype != torch.float32:
            assert torch.equal(p.detach(), masters[i].to(p.dtype))
    for got, want, k in ((opt.split(m), ref.m, 4), (opt.split(v), ref.v, 8)):
        for a, b in zip(got, want):
            if opt.state_bits == 8:
                assert torch.equal(a, b.float())
            elif a.numel():
                # v: 4 roundings a step, all of one sign; m's parts may cancel, and old errors fade by b1
                assert float(((a.double() - b).abs() - k * drift * U * (b.abs() + b.abs().max())).max()) <= 0


ref_size = None


def run(opt, ref, sizes, dtype, steps, seed, missing=()):
    global ref_size
    ref_size = [torch.zeros_like(w) for w in ref.w]
    for s in range(steps):
        grads = make(sizes, dtype, seed + s, 10.0 ** (-s % 3))
        grads = [None if (i, s) in missing else g.view_as(p) for i, (g, p) in enumerate(zip(grads, opt.params))]
        for p, g in zip(opt.params, grads):
            p.grad = g
        opt.step()
        ref.step(grads)
        # what a step's error in m (relative to its parts) does to the weights of later ones: the sizes add up
        ref_size = [a + b for a, b in zip(ref_size, ref.size)]
        compare(opt, ref, s + 1)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("max_norm", [None, 0.5, 1e9])
def test_steps_of_many_sizes(dtype, bits, max_norm):
    from checkers_mcts_amd import optim
    params = [p.requires_grad_(True) for p in make(SIZES, dtype, 1)]
    opt = optim.AdamW(params, lr=3e-3, betas=(0.9, 0.99), eps=1e-6, weight_decay=0.1, state_bits=bits, max_norm=max_norm, seed=12345678901234567)
    ref = Reference(opt, 3e-3, 0.1, (0.9, 0.99), 1e-6, bits, 12345678901234567, max_norm)
    run(opt, ref, SIZES, dtype, 4, 10)
    if max_norm is not None:
        assert opt.grad_norm.dtype == torch.float64 and abs(float(opt.grad_norm) - ref.norm) <= 1e-12 * ref.norm
    else:
        assert opt.grad_norm is None
    assert opt.steps.tolist() == [4] * len(SIZES)


@pytest.mark.parametrize("bits", [32, 8])
def test_more_tensors_than_a_launch_takes_and_missing_gradients(bits):
    from checkers_mcts_amd import optim
    sizes = [(37 * i) % 301 + 1 for i in range(230)]
    params = [p.requires_grad_(True) for p in make(sizes, torch.float32, 2)]
    opt = optim.AdamW(params, lr=1e-2, state_bits=bits, max_norm=2.0, eps=1e-7, seed=9)
    ref = Reference(opt, 1e-2, 1e-2, (0.9, 0.999), 1e-7, bits, 9, 2.0)
    missing = {(i, s) for i in range(230) for s in range(3) if (i + s) % 3 == 0 or 90 <= i < 200 and s == 1}
    run(opt, ref, sizes, torch.float32, 3, 20, missing)
    assert opt.steps.tolist() == ref.t


def test_no_gradient_at_all_changes_nothing():
    from checkers_mcts_amd import optim
    for max_norm in (None, 1.0):
        p = torch.ones(300, device="cuda", requires_grad=True)
        opt = optim.AdamW([p, torch.zeros((0, 4), device="cuda", requires_grad=True)], max_norm=max_norm)
        opt.step()
        assert (p == 1).all() and opt.steps.sum() == 0 and (opt.moments()[0] == 0).all()
        if max_norm:
            assert opt.grad_norm == 0
        p.grad = torch.zeros_like(p)
        opt.step()
        assert float((p - (1 - 1e-5)).abs().max()) <= 2 * U and opt.steps.tolist() == [1]     # the decay alone


@pytest.mark.parametrize("bits", [32, 8])
def test_groups_types_and_learning_rates_on_the_device(bits):
    from checkers_mcts_amd import optim
    a = [p.requires_grad_(True) for p in make((300, 5), torch.float32, 1) + make((129,), torch.bfloat16, 2)]
    b = [p.requires_grad_(True) for p in make((64,), torch.float16, 3) + make((1000,), torch.float32, 4)]
    lr = torch.tensor(0.01, device="cuda")
    opt = optim.AdamW([{"params": a, "weight_decay": 0.2}, {"params": b, "lr": lr, "betas": (0.5, 0.9), "eps": 1e-4}], lr=1e-3, state_bits=bits, max_norm=1.0, seed=4)
    refs = [Reference(opt, 1e-3, 0.2, (0.9, 0.999), 1e-8, bits, 4), Reference(opt, 0.01, 0.01, (0.5, 0.9), 1e-4, bits, 4)]
    for s in range(3):
        lr.fill_(0.01 * (s + 1))
        refs[1].lr = float(lr)
        grads = [torch.randn(p.shape, generator=torch.Generator(device="cuda").manual_seed(s), device="cuda").to(p.dtype) for p in a + b]
        for p, g in zip(a + b, grads):
            p.grad = g
        opt.step()
        norm = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
        assert abs(float(opt.grad_norm) - norm) <= 1e-12 * norm
        c = min(1.0, 1.0 / (norm + 1e-6))
        for r in refs:
            r.step([g.double() * c for g in grads])
        m, _ = opt.moments()
        masters = opt.split(opt.master)
        for i, p in enumerate(opt.params):
            r = refs[0] if i < 3 else refs[1]
            got = (p if p.dtype == torch.float32 else masters[i]).detach().double()
            assert float(((got - r.w[i]).abs() - 3 * (s + 1) * U * (r.size[i] + r.w[i].abs())).max()) <= 0
            if p.dtype != torch.float32:
                assert torch.equal(p.detach(), masters[i].to(p.dtype))
            if bits == 8:
                assert torch.equal(opt.split(m)[i], r.m[i].float())


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("shift", [0, 1, 3, 5])
def test_parameters_and_gradients_that_start_anywhere_and_what_lies_around_them(dtype, bits, shift):
    from checkers_mcts_amd import optim
    n = 4099
    buf = torch.full((n + 40,), 7.0, device="cuda", dtype=dtype)
    gbuf = torch.full((n + 40,), math.nan, device="cuda", dtype=dtype)
    p = buf[shift:shift + n].detach().requires_grad_(True)
    g = gbuf[shift + 2:shift + 2 + n]
    with torch.no_grad():
        p.copy_(make((n,), dtype, 5)[0])
    opt = optim.AdamW([p], state_bits=bits, seed=1, eps=1e-6)
    ref = Reference(opt, 1e-3, 1e-2, (0.9, 0.999), 1e-6, bits, 1)
    for s in range(2):
        g.copy_(make((n,), dtype, 6 + s)[0])
        p.grad = g
        opt.step()
        ref.step([g])
    got = (p if dtype == torch.float32 else opt.master[:n]).detach().double()
    assert float(((got - ref.w[0]).abs() - 2 * U * (ref.size[0] + 2 * ref.w[0].abs())).max()) <= 0
    assert (buf[:shift] == 7).all() and (buf[shift + n:] == 7).all() and gbuf[:shift + 2].isnan().all()
    if bits == 32:
        assert (opt.exp_avg[n:] == 0).all() and (opt.exp_avg_sq[n:] == 0).all()


def test_orders_of_dimensions():
    from checkers_mcts_amd import optim
    w = torch.randn((16, 8, 3, 3), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    one = w.clone().requires_grad_(True)
    two = w.clone().to(memory_format=torch.channels_last).requires_grad_(True)
    three = w.clone().permute(3, 1, 0, 2).contiguous().permute(2, 1, 3, 0).detach().requires_grad_(True)
    g = torch.randn_like(w)
    opt = [optim.AdamW([p]) for p in (one, two, three)]
    for p, o in zip((one, two, three), opt):
        p.grad = g                                                    # contiguous: copied for the others
        o.step()
        p.grad = g.to(memory_format=torch.channels_last)
        o.step()
    assert torch.equal(one, two) and torch.equal(one, three) and two.stride() != one.stride()
    assert torch.equal(opt[0].split(opt[0].moments()[0])[0], opt[1].split(opt[1].moments()[0])[0])
    tall = torch.zeros((5, 1), device="cuda").t().detach().requires_grad_(True)      # strides of dimensions of one element do not matter
    o = optim.AdamW([tall])
    tall.grad = torch.ones((1, 5), device="cuda")
    o.step()
    assert (tall < 0).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_gradients_that_are_not_finite(bits):
    from checkers_mcts_amd import optim
    p = torch.ones(1000, device="cuda", requires_grad=True)
    q = torch.ones(200, device="cuda", requires_grad=True)
    opt = optim.AdamW([p, q], state_bits=bits)
    p.grad, q.grad = torch.ones_like(p), torch.ones_like(q)
    p.grad[300] = math.nan
    p.grad[500] = math.inf
    opt.step()
    m, v = opt.split(opt.moments()[0]), opt.split(opt.moments()[1])
    assert p[300].isnan() and p[500].isnan() and int(p.isnan().sum()) == 2 and not q.isnan().any()
    if bits == 32:
        assert m[0][300].isnan() and m[0][500].isinf() and int(m[0].isfinite().sum()) == 998
    else:                                                             # a block's scale says that something in it is not finite
        assert m[0][256:512].isnan().all() and v[0][256:512].isnan().all() and m[0][:256].isfinite().all() and m[0][512:].isfinite().all()
    assert m[1].isfinite().all()
    for bad in (math.nan, math.inf):
        p = torch.ones(100, device="cuda", requires_grad=True)
        opt = optim.AdamW([p], state_bits=bits, max_norm=1.0)
        p.grad = torch.ones_like(p)
        p.grad[3] = bad
        opt.step()
        assert not math.isfinite(float(opt.grad_norm))
        assert p[3].isnan() and (p.isnan().all() if math.isnan(bad) else int(p.isnan().sum()) == 1)


@pytest.mark.parametrize("size", [1e-30, 1e-12, 1e15])
def test_very_small_and_large_gradients_in_8_bits(size):
    from checkers_mcts_amd import optim
    p = torch.zeros(512, device="cuda", requires_grad=True)
    opt = optim.AdamW([p], state_bits=8, seed=3, weight_decay=0.0, eps=1e-30)
    ref = Reference(opt, 1e-3, 0.0, (0.9, 0.999), 1e-30, 8, 3)
    for s in range(3):
        g = make((512,), torch.float32, s, size)[0]
        g[100:200] *= 1e-3
        g[200:210] = 0
        p.grad = g
        opt.step()
        ref.step([g])
        for got, want in zip(opt.moments(), (ref.m[0], ref.v[0])):
            assert torch.equal(got, want.float())
    if size > 1e-20:                                                  # (below, v falls out of float32: its root is that of 0)
        assert float(((p.detach().double() - ref.w[0]).abs() - 16 * 3 * U * (ref.size[0] + 3e-3)).max()) <= 0


def test_a_block_that_only_holds_tiny_values_beside_a_large_one():
    from checkers_mcts_amd import optim
    p = torch.zeros(128, device="cuda", requires_grad=True)
    opt = optim.AdamW([p], state_bits=8, seed=3)
    p.grad = torch.full((128,), 1e-6, device="cuda")
    p.grad[0] = 1e6
    opt.step()
    m, v = opt.moments()
    assert (m[1:] == 0).all() and (v[1:] > 0).all()                   # v is raised to the smallest code: a small m never meets eps alone
    before = p.detach().clone()
    opt.step()
    assert float((p.detach() - before)[1:].abs().max()) < 1e-3


@pytest.mark.parametrize("value", [1.0, 1.03, 0.77])
def test_the_rounding_is_right_on_average(value):
    """A moment of (1 - b) g for 65536 elements: the codes around it are taken so often that their mean is it, within 5 standard errors."""
    from checkers_mcts_amd import optim
    n = 65536
    p = torch.zeros(n, device="cuda", requires_grad=True)
    opt = optim.AdamW([p], state_bits=8, seed=77)
    p.grad = torch.full((n,), value, device="cuda")
    opt.step()
    for got, want in zip(opt.moments(), (0.1 * float(p.grad[0].double()), 0.001 * float(p.grad[0].double()) ** 2)):
        step = 2.0 ** (math.floor(math.log2(want)) - 3)
        low = math.floor(want / step) * step
        assert set(got.unique().tolist()) <= {low, low + step}
        f = (want - low) / step
        assert abs(float(got.double().mean()) - want) <= 5 * step * math.sqrt(f * (1 - f) / n) + step * 2.0 ** -16


def test_second_moments_follow_their_average():
    """v starts at 4 times g^2 and has to fall: after T steps of b2 = 0.99 its mean is g^2 (1 + 3 b2^T).  Each step's rounding has a variance of at
    most |v' - v| step <= 0.01 * 3 g^2 * g^2 / 2; together at most that / (1 - b2^2), over 8192 elements: 5 standard errors are 5 g^2 * sqrt(0.015 / 0.02 / 8192)."""
    from checkers_mcts_amd import optim
    n, T = 8192, 300
    p = torch.zeros(n, device="cuda", requires_grad=True)
    opt = optim.AdamW([p], state_bits=8, betas=(0.9, 0.99), seed=5)
    opt.load_moments(torch.zeros(n, device="cuda"), torch.full((n,), 4.0, device="cuda"), 1000)
    p.grad = torch.ones(n, device="cuda")
    for _ in range(T):
        opt.step()
    want = 1 + 3 * 0.99 ** T
    assert abs(float(opt.moments()[1].double().mean()) - want) <= 5 * math.sqrt(0.015 / 0.0199 / n)
    assert abs(float(opt.moments()[0].double().mean()) - 1.0) <= 5 * math.sqrt(0.1 / 8 / (1 - 0.81) / n) + 0.9 ** T


def test_seeds_repeat_and_differ():
    from checkers_mcts_amd import optim
    got = []
    for seed in (1, 1, 2, 1 << 40):
        p = torch.zeros(4096, device="cuda", requires_grad=True)
        opt = optim.AdamW([p], state_bits=8, seed=seed)
        for s in range(3):
            p.grad = make((4096,), torch.float32, s)[0]
            opt.step()
        got.append((p.detach().clone(), opt.exp_avg.clone(), opt.exp_avg_sq.clone()))
    assert all(torch.equal(a, b) for a, b in zip(got[0], got[1]))
    assert not torch.equal(got[0][2], got[2][2]) and not torch.equal(got[0][2], got[3][2])


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("bits", [32, 8])
def test_a_captured_step_replays_like_eager_ones(dtype, bits):
    from checkers_mcts_amd import optim
    sizes = (5, 3001, 128)

    def fresh():
        ps = [p.requires_grad_(True) for p in make(sizes, dtype, 3)]
        for p in ps:
            p.grad = torch.zeros_like(p)
        lr = torch.tensor(1e-3, device="cuda")
        return ps, lr, optim.AdamW(ps, lr=lr, state_bits=bits, max_norm=1.0, seed=6)

    def feed(ps, lr, s):
        lr.fill_(1e-3 * (s + 1))
        for p, g in zip(ps, make(sizes, dtype, 50 + s)):
            p.grad.copy_(g)
    ps, lr, opt = fresh()
    qs, lq, eager = fresh()
    feed(ps, lr, 0); feed(qs, lq, 0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        opt.step()
    torch.cuda.current_stream().wait_stream(side)
    eager.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for s in range(1, 5):
        feed(ps, lr, s); feed(qs, lq, s)
        torch.cuda.synchronize()
        graph.replay()
        eager.step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(ps, qs)) and torch.equal(opt.exp_avg, eager.exp_avg) and torch.equal(opt.exp_avg_sq, eager.exp_avg_sq)
        assert opt.steps.tolist() == eager.steps.tolist() == [s + 1] * 3 and torch.equal(opt.grad_norm, eager.grad_norm)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("bits", [32, 8])
def test_a_checkpoint_goes_on_where_it_was_left(dtype, bits, tmp_path):
    from checkers_mcts_amd import optim
    sizes = (100, 4000)
    ps = [p.requires_grad_(True) for p in make(sizes, dtype, 3)]
    opt = optim.AdamW(ps, lr=1e-2, state_bits=bits, seed=8)

    def step(ps, opt, s):
        for p, g in zip(ps, make(sizes, dtype, 90 + s)):
            p.grad = g
        opt.step()
    for s in range(2):
        step(ps, opt, s)
    torch.save({"opt": opt.state_dict(), "ps": [p.detach() for p in ps]}, tmp_path / "c.pt")
    saved = torch.load(tmp_path / "c.pt", weights_only=True)
    qs = [p.requires_grad_(True) for p in saved["ps"]]
    other = optim.AdamW(qs, lr=5.0, state_bits=bits)
    other.load_state_dict(saved["opt"])
    for s in range(2, 4):
        step(ps, opt, s); step(qs, other, s)
    assert all(torch.equal(p, q) for p, q in zip(ps, qs)) and torch.equal(opt.exp_avg_sq, other.exp_avg_sq)
    for bad in (optim.AdamW(qs, state_bits=40 - bits), optim.AdamW(qs[:1], state_bits=bits)):
        with pytest.raises(ValueError):
            bad.load_state_dict(saved["opt"])


@pytest.mark.parametrize("bits", [32, 8])
def test_moments_in_and_out(bits):
    from checkers_mcts_amd import optim
    shapes = ((3, 5), (1000,), (2, 64))
    ps = [torch.zeros(s, device="cuda", requires_grad=True) for s in shapes]
    opt = optim.AdamW(ps, state_bits=bits)
    g = torch.Generator(device="cuda").manual_seed(1)
    m = [torch.randn(s, generator=g, device="cuda") * 0.1 for s in shapes]
    v = [torch.rand(s, generator=g, device="cuda") * 0.01 for s in shapes]
    opt.load_moments(m, v, 17)
    assert opt.steps.tolist() == [17] * 3
    for got, want in zip((opt.split(opt.moments()[0]), opt.split(opt.moments()[1])), (m, v)):
        for a, b in zip(got, want):
            if bits == 32:
                assert torch.equal(a, b)
            else:                                                     # to nearest: half of an eighth at most, but for what is below the smallest code
                assert float(((a - b).abs() / b.abs().clamp(min=float(b.abs().max()) * 2.0 ** -14)).max()) <= 2.0 ** -4 * (1 + 2.0 ** -15)
    again = [t.clone() for t in opt.moments()]
    opt.load_moments(*again, 17)                                      # what codes hold comes back as it is
    assert all(torch.equal(a, b) for a, b in zip(opt.moments(), again))
    with pytest.raises(ValueError):
        opt.load_moments(m[:2], v, 1)
    with pytest.raises(ValueError):
        opt.load_moments(again[0][:5], again[1], 1)


def test_moments_of_steps_come_back_as_they_are():
    """Blocks whose largest value was rounded up to the next power of two, and what lies 14 powers below it, too."""
    from checkers_mcts_amd import optim
    n = 128 * 600
    for seed in range(3):
        p = torch.zeros(n, device="cuda", requires_grad=True)
        opt = optim.AdamW([p], state_bits=8, seed=seed)
        g = torch.Generator(device="cuda").manual_seed(seed)
        p.grad = (1.9 + 0.1 * torch.rand((n,), generator=g, device="cuda")) * 2.0 ** -torch.randint(0, 18, (n,), generator=g, device="cuda").float()
        opt.step()
        before = [t.clone() for t in opt.moments()]
        other = optim.AdamW([p], state_bits=8)
        other.load_moments(*before, 1)
        assert all(torch.equal(a, b) for a, b in zip(other.moments(), before))


def test_refusals():
    from checkers_mcts_amd import optim
    p = torch.zeros(100, device="cuda", requires_grad=True)
    for kw in (dict(state_bits=16), dict(max_norm=0.0), dict(max_norm=math.inf), dict(lr=-1.0), dict(lr=math.nan), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=0.0),
               dict(eps=-1e-8), dict(weight_decay=-0.1), dict(lr=torch.tensor(0.1)), dict(lr=torch.tensor(0.1, device="cuda", dtype=torch.float64))):
        with pytest.raises(ValueError):
            optim.AdamW([p], **kw)
    for bad in ([], [p, p], [{"params": [p]}, {"params": [p]}], [p, p.detach()[50:]], p, [torch.zeros(5, requires_grad=True)], [torch.zeros(5, device="cuda", dtype=torch.float64)],
                [torch.zeros(10, 10, device="cuda")[:, :5]], [torch.zeros(5, device="cuda").expand(3, 5)], [p * 2]):
        with pytest.raises(ValueError):
            optim.AdamW(bad)
    opt = optim.AdamW([p])
    p.grad = torch.sparse_coo_tensor(torch.tensor([[1]], device="cuda"), torch.ones(1, device="cuda"), (100,))
    with pytest.raises((ValueError, RuntimeError)):
        opt.step()
    p.grad = torch.ones(100, device="cuda")
    p.data = torch.zeros(50, device="cuda")
    with pytest.raises(ValueError):
        opt.step()


def test_parameters_changed_otherwise_than_by_a_step():
    from checkers_mcts_amd import optim
    p = torch.ones(100, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    opt = optim.AdamW([p], lr=0.0)
    p.grad = torch.zeros_like(p)
    with torch.no_grad():
        p.fill_(3.0)
    opt.reset_master()
    opt.step()
    assert (p == 3).all() and (opt.master[:100] == 3).all()
    # other memory of the same layout is taken over; the old one is left alone
    q = torch.ones(100, device="cuda", requires_grad=True)
    opt = optim.AdamW([q], lr=0.5, weight_decay=0.0, max_norm=1.0)
    q.grad = torch.ones_like(q)
    old = q.data
    q.data = torch.full((100,), 5.0, device="cuda")
    opt.step()
    assert (old == 1).all() and (q < 5).all()
    with pytest.raises(AttributeError):
        opt.max_norm = 2.0
    for change in (lambda t: t.half(), lambda t: t[:50], lambda t: t.cpu(), lambda t: t.reshape(10, 10)):
        r = torch.ones(100, device="cuda", requires_grad=True)
        opt = optim.AdamW([r])
        r.grad = torch.ones_like(r)
        r.data = change(r.data.clone())
        with pytest.raises(ValueError):
            opt.step()


def test_the_same_memory_in_another_order_is_refused():
    from checkers_mcts_amd import optim
    p = torch.ones((8, 8), device="cuda", requires_grad=True)
    opt = optim.AdamW([p])
    p.data = p.data.t()
    p.grad = torch.ones_like(p)
    assert p.grad.stride() == p.stride() == (1, 8)
    with pytest.raises(ValueError):
        opt.step()
    assert (p == 1).all() and int(opt.steps[0]) == 0


@pytest.mark.parametrize("bits", [32, 8])
def test_offsets_beyond_32_bits(bits):
    from checkers_mcts_amd import optim
    n, lead = 2 ** 31 + 300, 200
    small = torch.zeros(lead, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    p = torch.zeros(n, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    last = torch.ones(77, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    opt = optim.AdamW([small, p, last], lr=1e-2, state_bits=bits, max_norm=1e6, seed=3, weight_decay=0.0, eps=1e-6)
    assert opt.offsets == [0, 256, 256 + (n + 127) // 128 * 128]
    p.grad = torch.zeros_like(p)
    g = torch.randn(5000, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").bfloat16()
    p.grad[:5000] = g
    p.grad[-5000:] = g
    last.grad = g[:77].clone()
    opt.step()
    assert abs(float(opt.grad_norm) - math.sqrt(float(2 * g.double().square().sum() + g[:77].double().square().sum()))) <= 1e-9
    x = g.double()
    want = -0.01 * x / (x.abs() + 1e-6)
    for part in (p[:5000], p[-5000:]):
        assert float((part.detach().double() - want).abs().max()) <= 0.01 * 2.0 ** -8 * 1.01
    assert (p[5000:-5000] == 0).all() and (small == 0).all() and opt.steps.tolist() == [0, 1, 1]
    assert float((last.detach().double() - 1 - want[:77]).abs().max()) <= 2.0 ** -8 * 1.02
    if bits == 8:
        # the tensor's last whole block of 128, and the tensor behind it
        at = 256 + n // 128 * 128 - 128
        m, v = (t[at - (at - 256) % 128:][:128] for t in opt.moments())
        block = p.grad[n // 128 * 128 - 128:n // 128 * 128].double()
        rm, rv = dithers(3, at, 128, 1)
        assert torch.equal(m, rounded((1 - 0.9) * block, 16, rm, False).float())
        assert torch.equal(v, rounded((1 - 0.999) * block * block, 32, rv, True).float())


def test_the_step_counts_as_a_change_in_place():
    from checkers_mcts_amd import optim
    p = torch.ones(10, device="cuda", requires_grad=True)
    opt = optim.AdamW([p])
    loss = (p * p).sum()
    p.grad = torch.ones_like(p)
    opt.step()
    with pytest.raises(RuntimeError, match="inplace"):
        loss.backward()
    p.grad = torch.ones_like(p)
    opt.zero_grad(set_to_none=False)
    assert (p.grad == 0).all()
    opt.zero_grad()
    assert p.grad is None


def test_one_training_step_of_both_operators_and_a_second_one_captured():
    """Played moves with weights, an entropy term, clipping and 8-bit moments on a linear policy: against float64 throughout."""
    from checkers_mcts_amd import optim, policy
    n, f, v = 96, 40, 512
    g = torch.Generator(device="cuda").manual_seed(11)
    x = torch.randn((n, f), generator=g, device="cuda")
    W0 = torch.randn((v, f), generator=g, device="cuda") * 0.1
    b0 = torch.zeros((v,), device="cuda")
    move = torch.randint(0, v, (n,), generator=g, device="cuda")
    adv = torch.randn((n,), generator=g, device="cuda") / n
    legal = torch.rand((n, v), generator=g, device="cuda") < 0.05
    legal[torch.arange(n, device="cuda"), move] = True
    legal[5] = False
    adv[5] = 0.0

    def loss_of(W, b):
        out = policy.action_logprobs(x @ W.t() + b, move, mask=legal)
        return -(out.logp.clamp(min=-1e30) * adv).sum() - 0.01 * out.entropy.mean()
    W, b = W0.clone().requires_grad_(True), b0.clone().requires_grad_(True)
    opt = optim.AdamW([{"params": [W]}, {"params": [b], "weight_decay": 0.0}], lr=1e-3, state_bits=8, max_norm=0.05, eps=1e-7, seed=2)
    loss_of(W, b).backward()
    grads = [W.grad.clone(), b.grad.clone()]
    # the gradient in float64
    xd, Wd = x.double(), W0.double().requires_grad_(True)
    bd = b0.double().requires_grad_(True)
    z = (xd @ Wd.t() + bd).masked_fill(~legal, -math.inf)
    rows = torch.arange(n, device="cuda") != 5
    lp = torch.log_softmax(z[rows], 1)
    H = -(lp.exp() * lp.masked_fill(~legal[rows], 0.0)).sum(1)
    total = -(lp.gather(1, move[rows][:, None])[:, 0] * adv[rows].double()).sum() - 0.01 * H.sum() / n
    want = torch.autograd.grad(total, (Wd, bd))
    for got, w in zip(grads, want):
        # x W^T in float32 moves a logit by up to 40 products' roundings; then the operator's own, then the sum over 96 rows
        assert float((got.double() - w).abs().max()) <= 200 * U * float(w.abs().max() + 0.05)
    ref = [Reference(opt, 1e-3, 0.01, (0.9, 0.999), 1e-7, 8, 2, 0.05), Reference(opt, 1e-3, 0.0, (0.9, 0.999), 1e-7, 8, 2, 0.05)]
    for r in ref:
        r.step(grads)
    opt.step()
    for i, p in enumerate((W, b)):
        assert float(((p.detach().double() - ref[i].w[i]).abs() - U * (ref[i].size[i] + 2 * ref[i].w[i].abs() + 1e-9)).max()) <= 0
        assert torch.equal(opt.split(opt.moments()[0])[i], ref[i].m[i].float())


@pytest.mark.parametrize("optimizer", ["adamw", "adamw8"])
def test_train_nn_with_these_operators(optimizer, tmp_path, monkeypatch):
    import numpy as np
    from checkers_mcts_amd import policy, train
    from test_train_hip_gpu import make_batch
    monkeypatch.chdir(tmp_path)
    x, pi, tv = make_batch(400, 6)
    legal = policy.legal_from_features(x)
    some = legal.any(1)                                               # positions of a game that goes on, visits on their moves only
    x, tv, pi = x[some].contiguous(), tv[some].contiguous(), (pi + 1e-3)[some] * legal[some]
    pi = (pi / pi.sum(1, keepdim=True)).contiguous()
    data = train.TrainingData(dense=(x, pi, tv))
    kw = dict(PATIENCE=5, MIN_DELTA=0, VAL_SPLIT=0.2, TRAINING_ITERATION=0, BATCH_SIZE=32, CLR_SS_COEFF=4, NN_BASE_LR=1e-4, NN_MAX_LR=1e-3, EPOCHS=2, NUM_KERNELS=32,
              CONV_REG=1e-4, DENSE_REG=1e-4, POLICY_LOSS_WEIGHT=1.0, VALUE_LOSS_WEIGHT=1.0, SEED=1, OPTIMIZER=optimizer, MAX_GRAD_NORM=1.0, ENTROPY_WEIGHT=0.01, POLICY_METRICS=True)
    got = []
    for graph in (True, False):
        net = train.create_nn(**kw)
        before = net.pol_fc.weight.detach().clone()
        history, _ = train.train_nn(data, net, **dict(kw, USE_GRAPH=graph))
        h = history.history
        assert len(h["loss"]) == 2 and len(h["val_policy_entropy"]) == len(h["val_move_logp"]) == len(h["val_move_top3"]) == 2
        assert all(np.isfinite(x).all() for x in h.values()) and 0 <= h["val_move_top3"][-1] <= 1 and h["val_move_logp"][-1] < 0
        assert not torch.equal(before, net.pol_fc.weight.detach().cpu())
        got.append(net)
    with pytest.raises(ValueError, match="TRAIN_BACKEND"):
        train.train_nn(data, train.create_nn(**dict(kw, NUM_KERNELS=128)), **dict(kw, TRAIN_BACKEND="hip"))


@pytest.mark.parametrize("native", [True, False])
def test_a_parameter_seen_otherwise_beside_the_gradient_it_had_is_refused(native, monkeypatch):
    from checkers_mcts_amd import optim
    if not native:                                                    # as on a torch without the native comparison
        monkeypatch.setattr(optim, "_make_guards", None)
    p = torch.arange(64.0, device="cuda").reshape(8, 8).requires_grad_(True)
    opt = optim.AdamW([p])
    p.grad = torch.arange(64.0, device="cuda").reshape(8, 8) - 30
    for _ in range(3):
        opt.step()
    assert native == (opt._guards is not None) or optim._make_guards is None
    before = p.detach().clone()
    p.data = p.data.t()
    for again in (False, True):
        if again:
            (p * 2.0).sum().backward()                                # autograd adds to the gradient that is there, in its order
        assert p.grad.stride() == (8, 1) and p.stride() == (1, 8)
        with pytest.raises(ValueError):
            opt.step()
        assert torch.equal(p.detach().t(), before) and int(opt.steps[0]) == 3
    p.data = p.data.t()                                               # as it was
    opt.step()
    assert int(opt.steps[0]) == 4


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("kept", [False, True])
def test_a_parameter_of_another_type_at_the_same_address_is_refused(kept, native, monkeypatch):
    from checkers_mcts_amd import optim
    if not native:
        monkeypatch.setattr(optim, "_make_guards", None)
    p = torch.ones(64, device="cuda", dtype=torch.bfloat16).requires_grad_(True)
    opt = optim.AdamW([p])
    p.grad = torch.ones_like(p)
    for _ in range(3):
        opt.step()
    p.data = p.data.view(torch.float16)
    if not kept:
        p.grad = torch.ones(64, device="cuda", dtype=torch.float16)
    before = p.detach().clone()
    with pytest.raises(ValueError):
        opt.step()
    assert torch.equal(p.detach(), before) and int(opt.steps[0]) == 3


@pytest.mark.skipif(not hasattr(torch.Tensor, "grad_dtype"), reason="gradients have their parameters' type")
def test_a_gradient_of_another_type_is_refused():
    from checkers_mcts_amd import optim
    p = torch.ones(64, device="cuda", dtype=torch.bfloat16).requires_grad_(True)
    opt = optim.AdamW([p])
    p.grad = torch.ones_like(p)
    for _ in range(3):
        opt.step()
    p.grad = None
    p.grad_dtype = torch.float16
    p.grad = torch.ones(64, device="cuda", dtype=torch.float16)
    with pytest.raises(ValueError):
        opt.step()
    assert int(opt.steps[0]) == 3


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("shape", [(), (1,), (1, 1)], ids=str)
def test_gradients_that_are_seen_negated(shape, native, monkeypatch):
    """The gradient of an imaginary part may come as a view of its conjugate: the memory holds the opposite sign."""
    from checkers_mcts_amd import optim
    if not native:
        monkeypatch.setattr(optim, "_make_guards", None)
    w, one = torch.zeros(shape, device="cuda", requires_grad=True), torch.ones(shape, device="cuda")
    opt = optim.AdamW([w], lr=0.5, weight_decay=0.0, max_norm=10.0)
    (torch.complex(one, w).conj() * torch.complex(one, 3 * one)).imag.sum().backward()   # (1 - i w) (1 + 3 i): 3 - w
    assert w.grad.is_neg() and float(w.grad) == -1
    opt.step()
    assert abs(float(w.detach()) - 0.5) <= 0.5 * (16 * U + 1e-8)               # 12 u of the update, 2 of w, and eps beside 1
    p = torch.complex(one, one).conj().imag.detach().requires_grad_(True)
    assert p.is_neg() and p.is_leaf
    with pytest.raises(ValueError, match="negative"):
        optim.AdamW([p])


def test_a_checkpoint_of_a_learning_rate_on_the_device(tmp_path):
    """Loading keeps the scalar that the caller fills and captured steps read; nothing is shared with the optimiser it came from."""
    from checkers_mcts_amd import optim
    scalar = lambda v: torch.tensor(v, device="cuda")

    def build(lr):
        ps = [p.requires_grad_(True) for p in make((300, 70), torch.float32, 3)]
        for p, g in zip(ps, make((300, 70), torch.float32, 4)):
            p.grad = g
        return ps, optim.AdamW(ps, lr=lr, weight_decay=0.0)
    ps, opt = build(scalar(1e-2))
    opt.step()
    qs, other = build(mine := scalar(5.0))
    other.load_state_dict(opt.state_dict())
    assert other.param_groups[0]["lr"] is mine and mine.data_ptr() != opt.param_groups[0]["lr"].data_ptr() and float(mine) == float(opt.param_groups[0]["lr"])
    mine.fill_(0.25)
    assert float(opt.param_groups[0]["lr"]) == float(scalar(1e-2))
    # a captured step goes on reading it
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other.step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        other.step()
    other.load_state_dict(opt.state_dict())                           # lr 1e-2 again
    with torch.no_grad():
        for p, q in zip(ps, qs):
            q.copy_(p)
    for _ in range(3):
        graph.replay()
        opt.step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(ps, qs))
    # from a file, mapped to the host; a number where the saved one is on the device, and the other way round
    torch.save(opt.state_dict(), tmp_path / "o.pt")
    saved = torch.load(tmp_path / "o.pt", map_location="cpu", weights_only=True)
    for lr in (scalar(3.0), 3.0):
        rs, third = build(lr)
        third.load_state_dict(saved)
        now = third.param_groups[0]["lr"]
        assert now.is_cuda and now.dtype == torch.float32 and float(now) == float(scalar(1e-2)) and torch.equal(third.exp_avg, opt.exp_avg)
        third.step()
    _, fourth = build(0.125)
    rs, third = build(mine := scalar(3.0))
    third.load_state_dict(fourth.state_dict())
    assert third.param_groups[0]["lr"] is mine and float(mine) == 0.125
    bad = opt.state_dict()
    bad["param_groups"][0]["lr"] = torch.ones(2)
    before = [t.clone() for t in (third.exp_avg, third.steps)]
    with pytest.raises(ValueError):
        third.load_state_dict(bad)
    assert torch.equal(before[0], third.exp_avg) and torch.equal(before[1], third.steps) and float(mine) == 0.125


def test_a_checkpoint_of_parameters_that_lie_otherwise_is_refused():
    """Moments are kept in the order of the parameters' memory, step counts in the order of groups and types."""
    from checkers_mcts_amd import optim
    param = lambda t: t.cuda().requires_grad_(True)
    conv = torch.arange(2.0 * 3 * 4 * 4).reshape(2, 3, 4, 4)

    def saved(params):
        opt = optim.AdamW(params)
        for p in opt.params:
            p.grad = torch.ones_like(p)
        opt.step()
        return opt.state_dict()
    there = conv.contiguous(memory_format=torch.channels_last)
    for one, other in ((conv, there), (there, conv), (there, conv.permute(1, 0, 2, 3).contiguous().permute(1, 0, 2, 3))):
        with pytest.raises(ValueError):
            optim.AdamW([param(one)]).load_state_dict(saved([param(other)]))
    for one, other in ((conv, conv.reshape(-1)), (there, there.clone()), (torch.ones(5, 6, 1, 1), torch.ones(5, 6, 1, 1).contiguous(memory_format=torch.channels_last))):
        optim.AdamW([param(one)]).load_state_dict(saved([param(other)]))
    # the same sizes, types in another order
    a, b = torch.ones(100), torch.ones(100).bfloat16()
    here = saved([param(a), param(b)])
    with pytest.raises(ValueError):
        optim.AdamW([param(b), param(a)]).load_state_dict(here)
    with pytest.raises(ValueError):
        optim.AdamW([param(a), param(torch.ones(100).half())]).load_state_dict(here)
    # the same tensors, divided into groups otherwise
    three = lambda: [param(torch.ones(100)) for _ in range(3)]
    groups = lambda ps, k: [{"params": ps[:k]}, {"params": ps[k:]}]
    here = saved(groups(three(), 1))
    with pytest.raises(ValueError):
        optim.AdamW(groups(three(), 2)).load_state_dict(here)
    other = optim.AdamW(groups(three(), 1))
    other.load_state_dict(here)
    assert other.steps.tolist() == [1, 1, 1]
    old = {k: v for k, v in here.items() if k != "layout"}            # saved before the layout was part of it
    other.load_state_dict(old)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("bits", [32, 8])
def test_what_else_changes_a_16_bit_parameter_is_not_undone(dtype, bits):
    """A module's weights loaded after the optimiser was made, or other memory with other values: the master copies follow where the
    parameter is no longer their rounding, and stay where it is."""
    from checkers_mcts_amd import optim
    a, b = (p.requires_grad_(True) for p in make((1000, 64), dtype, 3, 1.0))
    opt = optim.AdamW([a, b], lr=1e-4, weight_decay=0.0, state_bits=bits)
    for p, g in zip((a, b), make((1000, 64), dtype, 4)):
        p.grad = g
    opt.step()
    masters = [m.clone() for m in opt.split(opt.master)]
    assert not torch.equal(masters[0], a.detach().float())
    still = torch.zeros(1000, dtype=torch.bool, device="cuda")
    still[::2] = True
    new = torch.where(still, a.detach(), a.detach() + 1)
    assert bool((new != a)[~still].all())
    with torch.no_grad():
        a.copy_(new)
    for p in (a, b):
        p.grad = torch.zeros_like(p)
    for g in opt.param_groups:
        g["lr"] = 0.0
    opt.step()                                                        # of size zero
    assert torch.equal(a.detach(), new)
    now = opt.split(opt.master)
    assert torch.equal(now[0][still], masters[0][still]) and torch.equal(now[0][~still], new.float()[~still]) and torch.equal(now[1], masters[1])
    # other memory
    more = new + 2
    a.data = more.clone()
    opt.step()
    assert torch.equal(a.detach(), more) and torch.equal(opt.split(opt.master)[0], more.float()) and torch.equal(opt.split(opt.master)[1], masters[1])
    # without a gradient it is nobody's turn
    a.grad = None
    with torch.no_grad():
        a.fill_(7.0)
    opt.step()
    assert (a == 7).all()
    # the state of a checkpoint is the state: its masters are not taken from parameters that were changed before
    state = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in opt.state_dict().items()}
    state["master"].fill_(3.0)
    with torch.no_grad():
        b.fill_(9.0)
    opt.load_state_dict(state)
    b.grad = torch.zeros_like(b)
    opt.step()
    assert (b == 3).all()


def test_steps_of_16_bit_parameters_in_one_buffer_are_not_taken_for_changes(monkeypatch):
    """Views of one buffer share a version counter."""
    from checkers_mcts_amd import optim
    flat = torch.ones(300, device="cuda", dtype=torch.bfloat16)
    ps = [flat[i:i + 100].detach().requires_grad_(True) for i in (0, 100, 200)]
    opt = optim.AdamW(ps, lr=1e-4)
    for p in ps:
        p.grad = torch.ones_like(p)
    followed = []
    whole = opt._follow
    monkeypatch.setattr(opt, "_follow", lambda which: (followed.append(list(which)), whole(which)))
    for s in range(4):
        if s == 2:
            ps[1].grad = None
        opt.step()
    assert followed == [] and (opt.split(opt.master)[0] < 1).all()
    flat[250:].fill_(5.0)
    ps[2].grad = torch.zeros_like(ps[2])
    opt.step()
    assert followed == [[0, 1, 2]] and (ps[2].detach()[50:] > 4).all() and (ps[2].detach()[:50] < 1.01).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_a_captured_training_step_of_both_operators(bits):
    """Forward, loss, backward, clipping and step in one graph, replayed with new inputs between eager work of another optimiser: as eager steps."""
    from checkers_mcts_amd import optim, policy
    n, f, v = 64, 24, 512

    def batch(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        x, move = torch.randn((n, f), generator=g, device="cuda"), torch.randint(0, v, (n,), generator=g, device="cuda")
        legal = torch.rand((n, v), generator=g, device="cuda") < 0.05
        legal[torch.arange(n, device="cuda"), move] = True
        return x, move, legal

    def build():
        g = torch.Generator(device="cuda").manual_seed(0)
        W = (torch.randn((v, f), generator=g, device="cuda") * 0.1).requires_grad_(True)
        b = torch.zeros((v,), device="cuda").requires_grad_(True)
        return (W, b), optim.AdamW([{"params": [W]}, {"params": [b], "weight_decay": 0.0}], lr=1e-2, state_bits=bits, max_norm=0.05, seed=2)

    def train(params, opt, x, move, legal):
        opt.zero_grad(set_to_none=False)
        out = policy.action_logprobs(torch.addmm(params[1], x, params[0].t()), move, mask=legal, top=3)
        loss = -out.logp.mean() - 0.01 * out.entropy.mean()
        loss.backward()
        opt.step()
        return loss.detach(), out.top_action
    mine, opt = build()
    theirs, eager = build()
    static = [t.clone() for t in batch(100)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        train(mine, opt, *static)
    torch.cuda.current_stream().wait_stream(side)
    train(theirs, eager, *batch(100))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = train(mine, opt, *static)
    for rep in range(5):
        for t, new in zip(static, batch(101 + rep)):
            t.copy_(new)
        graph.replay()
        want = train(theirs, eager, *batch(101 + rep))                 # eager work between the replays
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(mine, theirs)) and torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert torch.equal(opt.exp_avg_sq, eager.exp_avg_sq) and opt.steps.tolist() == eager.steps.tolist() == [rep + 2] * 2
