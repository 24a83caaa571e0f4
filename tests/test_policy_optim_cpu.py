"""CPU: what policy.action_logprobs, optim.AdamW and their C entry points refuse, before anything reaches a GPU."""
import ctypes as C

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from checkers_mcts_amd import build, _lib
    build.build()
    return _lib.load()


def args(**kw):
    from checkers_mcts_amd import policy
    a = policy.LogprobsArgs(n=4, v=100, row_stride=100, dtype=0, inv_temperature=1.0)
    a.logits = a.entropy = a.logp = a.stats = a.grad = a.actions = 4096      # never read: every call here ends at a check
    a.action_bytes, a.grad_stride = 8, 100
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("bad", [dict(n=-1), dict(v=0), dict(v=(1 << 30) + 1), dict(n=(1 << 32) + 1), dict(dtype=3), dict(dtype=-1), dict(mask_kind=3), dict(mask_kind=1),
                                 dict(mask_kind=2, mask=4096), dict(n_given=65), dict(n_given=-1), dict(top=65), dict(n_given=1, action_bytes=2),
                                 dict(n_given=1, actions=None), dict(inv_temperature=0.0), dict(inv_temperature=float("inf")), dict(inv_temperature=float("nan")),
                                 dict(inv_temperature=-1.0), dict(row_stride=-1), dict(logits=None), dict(mask_kind=1, mask=4096, mask_stride=-1)], ids=str)
def test_bad_arguments_of_logprobs(lib, bad):
    for fn in (lib.ckr_logprobs_forward, lib.ckr_logprobs_backward):
        assert fn(C.byref(args(**bad)), None) == -1
        assert b"ckr_logprobs" in lib.ckr_last_error()
    assert lib.ckr_logprobs_scratch(C.byref(args(**bad))) == -1


def test_missing_outputs_and_null_structures(lib):
    assert lib.ckr_logprobs_forward(None, None) == -1 and lib.ckr_logprobs_backward(None, None) == -1 and lib.ckr_logprobs_scratch(None) == -1
    assert lib.ckr_logprobs_forward(C.byref(args(entropy=None)), None) == -1
    assert lib.ckr_logprobs_forward(C.byref(args(n_given=1, logp=None)), None) == -1
    assert lib.ckr_logprobs_forward(C.byref(args(top=2)), None) == -1
    assert lib.ckr_logprobs_backward(C.byref(args(stats=None)), None) == -1
    assert lib.ckr_logprobs_backward(C.byref(args(grad=None)), None) == -1
    assert lib.ckr_logprobs_backward(C.byref(args(grad_stride=99)), None) == -1
    assert lib.ckr_logprobs_backward(C.byref(args(n_given=1)), None) == -1


def test_scratch_memory_and_alignment(lib):
    few = args(n=2, v=1 << 20, row_stride=1 << 20, top=3, top_action=4096, top_logp=4096)
    need = lib.ckr_logprobs_scratch(C.byref(few))
    assert need > 0 and lib.ckr_logprobs_scratch(C.byref(args(n=1 << 16, v=1 << 20))) == 0 and lib.ckr_logprobs_scratch(C.byref(args(v=1))) == 0
    assert lib.ckr_logprobs_forward(C.byref(few), None) == -1 and b"scratch" in lib.ckr_last_error()
    few.scratch, few.scratch_bytes = 4096, need - 1
    assert lib.ckr_logprobs_forward(C.byref(few), None) == -1
    for odd in (dict(stats=4100), dict(scratch=4104)):
        assert lib.ckr_logprobs_forward(C.byref(args(**odd)), None) == -1


def test_no_cpu_fallback(lib):
    if torch.cuda.is_available():
        pytest.skip("GPU present")
    assert lib.ckr_logprobs_forward(C.byref(args()), None) == -2
    assert b"no CPU fallback" in lib.ckr_last_error()
    from checkers_mcts_amd import optim, policy
    with pytest.raises(ValueError, match="cuda"):
        policy.action_logprobs(torch.zeros(2, 5))
    with pytest.raises(ValueError, match="on one GPU"):
        optim.AdamW([torch.zeros(4, requires_grad=True)])


def adamw_args(n=2, **kw):
    from checkers_mcts_amd import optim
    keep = {"sizes": (C.c_int64 * n)(*[10] * n), "offsets": (C.c_int64 * n)(*[128 * i for i in range(n)]),
            "params": (C.c_void_p * n)(*[4096] * n), "grads": (C.c_void_p * n)(*[4096] * n)}
    a = optim.AdamWArgs(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, count=n, state_bits=32)
    a.m = a.v = a.d_step = a.d_ticket = a.m_scale = a.v_scale = a.master = 4096
    keep.update({k: kw.pop(k) for k in list(kw) if k in keep})
    for k, v in keep.items():
        setattr(a, k, None if v is None else C.addressof(v))
    for k, v in kw.items():
        setattr(a, k, v)
    a._keep = keep
    return a


@pytest.mark.parametrize("bad", [dict(count=0), dict(sizes=None), dict(offsets=None), dict(params=None), dict(grads=None), dict(m=None), dict(v=None), dict(d_step=None),
                                 dict(d_ticket=None), dict(state_bits=16), dict(state_bits=8, m_scale=None), dict(dtype=1, master=None), dict(dtype=5), dict(beta1=1.0),
                                 dict(beta2=-0.1), dict(eps=0.0), dict(eps=float("nan")), dict(beta1=float("nan")), dict(sizes=(C.c_int64 * 2)(10, 0)),
                                 dict(sizes=(C.c_int64 * 2)(10, 1 << 37)), dict(offsets=(C.c_int64 * 2)(0, 64)), dict(offsets=(C.c_int64 * 2)(-128, 0)),
                                 dict(params=(C.c_void_p * 2)(4096, None))], ids=lambda b: ",".join(b))
def test_bad_arguments_of_adamw(lib, bad):
    assert lib.ckr_adamw_step(C.byref(adamw_args(**bad)), None) == -1
    assert b"ckr_adamw_step" in lib.ckr_last_error()


def test_bad_arguments_of_the_norm_and_the_moments(lib):
    sizes, grads, kinds = (C.c_int64 * 2)(10, 10), (C.c_void_p * 2)(4096, 4096), (C.c_int32 * 2)(0, 0)
    good = [2, C.addressof(sizes), C.addressof(grads), C.addressof(kinds), 1.0, 4096, 4096, 4096, 4096, None]
    for i, v in ((0, 0), (1, None), (2, None), (3, None), (4, 0.0), (4, -1.0), (4, float("nan")), (5, None), (6, 0), (7, None), (8, None)):
        bad = list(good)
        bad[i] = v
        assert lib.ckr_grad_norm(*bad) == -1, i
    kinds[1] = 7
    assert lib.ckr_grad_norm(*good) == -1
    for fn, good in ((lib.ckr_adamw_read_moments, [4096, 4096, 4096, 4096, 256, 4096, 4096, None]), (lib.ckr_adamw_write_moments, [4096, 4096, 256, 4096, 4096, 4096, 4096, None])):
        n = good.index(256)
        for i in range(7):
            bad = list(good)
            bad[i] = 100 if i == n else None
            assert fn(*bad) == -1
        bad[n] = 0
        assert fn(*bad) == -1


def test_train_nn_refuses_what_cannot_run_together():
    from checkers_mcts_amd import train
    data = [[torch.zeros(15, 8, 8).double().numpy(), torch.zeros(8, 8, 8).double().numpy() + 1 / 512, 0.0, 0.0]] * 4
    kw = dict(PATIENCE=1, MIN_DELTA=0, VAL_SPLIT=0, TRAINING_ITERATION=0, BATCH_SIZE=2, CLR_SS_COEFF=4, NN_BASE_LR=1e-3, NN_MAX_LR=1e-2, EPOCHS=1, NUM_KERNELS=8,
              CONV_REG=0.0, DENSE_REG=0.0, POLICY_LOSS_WEIGHT=1.0, VALUE_LOSS_WEIGHT=1.0, DEVICE="cpu", SEED=1)
    for more, word in ((dict(OPTIMIZER="sgd"), "OPTIMIZER"), (dict(OPTIMIZER="adamw"), "GPU"), (dict(ENTROPY_WEIGHT=0.1), "GPU"), (dict(POLICY_METRICS=True), "GPU"),
                       (dict(MAX_GRAD_NORM=1.0), "MAX_GRAD_NORM"), (dict(WEIGHT_DECAY=0.1), "WEIGHT_DECAY")):
        with pytest.raises(ValueError, match=word):
            train.train_nn(data, train.create_nn(**kw), **dict(kw, **more))


def stubbed(monkeypatch, calls):
    """policy's autograd function on host tensors: `calls` gets a copy of every structure that would have been launched."""
    from checkers_mcts_amd import policy
    monkeypatch.setattr(policy, "_call", lambda fn, a, device: calls(policy.LogprobsArgs.from_buffer_copy(a)))
    return lambda x, a, mask=None, top=0: policy._Logprobs.apply(x, a, mask, policy.MASK_NONE if mask is None else policy.MASK_BYTES, top, 1.0)


def test_two_backward_passes_of_one_graph_at_the_same_time(lib, monkeypatch):
    """Without autograd's own threads each caller runs the function itself: what one fills in is not another's."""
    import threading
    inside, seen = threading.Barrier(2, timeout=20), []

    def call(a):
        if a.grad:
            seen.append((a.grad, a.g_logp))
    from checkers_mcts_amd import policy
    x, a = torch.zeros(3, 7, requires_grad=True), torch.zeros((3, 2), dtype=torch.int64)
    apply = stubbed(monkeypatch, lambda a: None)
    logp, entropy, _, _ = apply(x, a)
    monkeypatch.setattr(policy, "_call", lambda fn, a, device: (inside.wait(), call(a), inside.wait()))       # both have filled theirs in before either is looked at
    gs, got, failed = [torch.full((3, 2), float(i)) for i in range(2)], [None, None], []

    def run(i):
        try:
            with torch.autograd.set_multithreading_enabled(False):
                got[i], = torch.autograd.grad(logp, x, gs[i], retain_graph=True)
        except Exception as e:
            failed.append(e)
    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not failed and len(seen) == 2
    assert {g for g, _ in seen} == {g.data_ptr() for g in got} and {g for _, g in seen} == {g.data_ptr() for g in gs}


@pytest.mark.parametrize("which", ["logits", "actions", "mask", "stats"])
@pytest.mark.parametrize("change", ["type", "shape", "device"])
def test_saved_tensors_that_come_back_as_others_are_refused(lib, monkeypatch, which, change):
    seen = []
    apply = stubbed(monkeypatch, seen.append)
    x, a, mask = torch.zeros(3, 7, requires_grad=True), torch.zeros((3, 2), dtype=torch.int64), torch.ones(3, 7, dtype=torch.bool)
    is_it = {"logits": lambda t: t.shape == (3, 7) and t.dtype == torch.float32, "actions": lambda t: t.dtype == torch.int64, "mask": lambda t: t.dtype == torch.bool,
             "stats": lambda t: t.shape == (3, 4)}[which]
    other = {"type": lambda t: t.to(torch.float64 if t.is_floating_point() else torch.int16), "shape": lambda t: t[:2], "device": lambda t: t.to("meta")}[change]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: other(t) if is_it(t) else t):
        logp, entropy, _, _ = apply(x, a, mask)
    forward = len(seen)
    with pytest.raises(RuntimeError, match="saved"):
        torch.autograd.grad((logp.sum() + entropy.sum()), x)
    assert len(seen) == forward                                        # nothing was launched


def test_saved_tensors_that_come_back_in_another_order_are_copied(lib, monkeypatch):
    seen = []
    apply = stubbed(monkeypatch, seen.append)
    x, a, mask = torch.zeros(3, 7, requires_grad=True), torch.zeros((3, 2), dtype=torch.int64), torch.ones(3, 7, dtype=torch.bool)
    keep = []

    def turned(t):
        keep.append(t.t().contiguous().t() if t.dim() == 2 else t)
        return keep[-1]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, turned):
        logp, entropy, _, _ = apply(x, a, mask)
    torch.autograd.grad((logp.sum() + entropy.sum()), x)
    addresses = {t.data_ptr() for t in keep}
    b = seen[-1]
    assert len(keep) == 4 and not addresses & {b.logits, b.actions, b.mask, b.stats} and (b.row_stride, b.mask_stride) == (7, 7)


def test_train_nn_takes_none_for_what_is_not_given(tmp_path, monkeypatch):
    from checkers_mcts_amd import train
    monkeypatch.chdir(tmp_path)
    data = [[torch.zeros(15, 8, 8).double().numpy(), torch.zeros(8, 8, 8).double().numpy() + 1 / 512, 0.0, 0.0]] * 4
    kw = dict(PATIENCE=1, MIN_DELTA=0, VAL_SPLIT=0, TRAINING_ITERATION=0, BATCH_SIZE=2, CLR_SS_COEFF=4, NN_BASE_LR=1e-3, NN_MAX_LR=1e-2, EPOCHS=1, NUM_KERNELS=8,
              CONV_REG=0.0, DENSE_REG=0.0, POLICY_LOSS_WEIGHT=1.0, VALUE_LOSS_WEIGHT=1.0, DEVICE="cpu", SEED=1, MODEL_SUFFIX=".pt",
              OPTIMIZER="adam", MAX_GRAD_NORM=None, WEIGHT_DECAY=None, ENTROPY_WEIGHT=None)
    history, _ = train.train_nn(data, train.create_nn(**kw), **kw)
    assert len(history.history["loss"]) == 1
