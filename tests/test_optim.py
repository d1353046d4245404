"""The optimizer operators: oracle pinned to torch and to its own definition on CPU, refusals, GPU parity.

Tolerances.  u = 2^-24 is the largest relative error of one 32-bit operation, and the constants b, 1 - b
are rounded to 32 bits too.  With c g the clipped gradient (its factor is off by at most 4 u):
    m = b1 m + (1 - b1) c g          off by at most   (2 + 1) u |b1 m| + (4 + 3 + 1) u |(1 - b1) c g|
    v = b2 v + (1 - b2) (c g)^2      off by at most   (2 + 1) u b2 v + (8 + 4 + 1) u (1 - b2) (c g)^2
    p = p d - rate m / (sqrt(v) root + eps)
        d: 1 u, product 1 u, difference 1 u                                  ->  4 u |p|
        rate, root: 4 u each (expm1f 1 ulp = 2 u, a division, a rounding), sqrt(v): half of v's plus 1 u,
        product, sum, two divisions, difference 1 u each                     ->  24 u |step| + the step that m's error makes
The tests allow these sums, plus half a spacing where a result is rounded to 16 bits.
"""
import ctypes
import math

import numpy as np
import pytest
import torch

from flexsae_b200 import _native as nv
from flexsae_b200 import optim
from oracle import optim_oracle as orc

U = 2.0 ** -24
HALF = {torch.float32: (0.0, 0.0), torch.bfloat16: (2.0 ** -8, 2.0 ** -134), torch.float16: (2.0 ** -11, 2.0 ** -25)}
gpu = pytest.mark.gpu


# ---- CPU: the oracle --------------------------------------------------------------------------------
def test_oracle_is_torchs_adamw():
    g = torch.Generator().manual_seed(0)
    p = torch.randn(40, 7, generator=g, dtype=torch.float64, requires_grad=True)
    opt = torch.optim.AdamW([p], lr=3e-3, betas=(0.8, 0.95), eps=1e-6, weight_decay=0.1)
    q, m, v = p.detach().numpy().copy(), np.zeros((40, 7)), np.zeros((40, 7))
    for t in range(1, 6):
        p.grad = torch.randn(40, 7, generator=g, dtype=torch.float64)
        opt.step()
        q, m, v = orc.adamw(q, p.grad.numpy(), m, v, t, 3e-3, (0.8, 0.95), 1e-6, 0.1)
        np.testing.assert_allclose(p.detach().numpy(), q, rtol=1e-12, atol=1e-14)


def test_oracle_keeps_rows_at_unit_length_and_steps_across_them():
    r = np.random.default_rng(0)
    w = r.standard_normal((5, 12))
    w /= np.linalg.norm(w, axis=1, keepdims=True)
    w[3] = 0
    p, m, _ = orc.adamw(w, r.standard_normal((5, 12)), np.zeros((5, 12)), np.zeros((5, 12)), 1, 1e-2, unit_rows=True)
    np.testing.assert_allclose(np.linalg.norm(p, axis=1), 1, rtol=1e-14)
    np.testing.assert_allclose(np.sum(m * w, axis=1), 0, atol=1e-15)         # the gradient across its row


@pytest.mark.parametrize("kind,dtype", [("m", torch.float8_e4m3fn), ("v", torch.float8_e5m2)])
def test_oracle_formats_are_torchs(kind, dtype):
    c = np.arange(256, dtype=np.uint8)
    if kind == "v":
        c = c[(c & 0x7F) < 0x7C]
    want = torch.from_numpy(c).view(dtype).float().numpy()
    np.testing.assert_array_equal(orc.widen(c, kind), want)


@pytest.mark.parametrize("kind,largest", [("m", 448.0), ("v", 57344.0)])
def test_oracle_rounding_is_right_on_average(kind, largest):
    """Every value goes to one of its two neighbours, upwards with the right probability: over all 2^k random
    numbers the mean is the value, up to the last bits that the random number has no room for (2^-20 of a spacing) and
    the rounding of x / scale (2 u)."""
    r = np.random.default_rng(1)
    x = (r.standard_normal(256) * 10.0 ** r.uniform(-6, 0, 256)).astype(np.float32)
    if kind == "v":
        x = np.abs(x)
    s = orc.scales(x, largest)
    bits = 20 if kind == "m" else 21
    grid = orc.E4M3 if kind == "m" else orc.E5M2
    y = np.abs(x.astype(np.float64) / s[0])
    if kind == "v":
        y = np.maximum(y, grid[1])
    lower = grid[np.searchsorted(grid, y, side="right") - 1]
    upper = grid[np.minimum(np.searchsorted(grid, y, side="right"), len(grid) - 1)]
    n = 1024
    total = np.zeros(256)
    for k in range(n):                              # random numbers spread evenly: the mean is exact to 1 / n of a spacing
        c = orc.codes(x, s, np.full(256, (k << bits) // n), kind)
        q = np.abs(orc.widen(c, kind).astype(np.float64))
        assert np.all((q == lower) | (q == upper))
        total += q
    assert np.all(np.abs(total / n - y) <= (upper - lower) / n + 2 * U * y)


def test_second_moment_follows_a_change_that_rounding_to_nearest_would_not_show():
    """The reason for the random rounding: gradients of size 1 for 100 steps, then of size 0.1 beside one of size
    1 that holds the scale.  After 3000 steps the average of v is 0.01 + (v0 - 0.01) * 0.999^3000, with v0 what the
    first codes stand for (cut off without random bits, 1 becomes the second largest code, 6/7); 2048 elements are
    averaged, each within about 75 % of it, so their mean is within 6 % (4 standard deviations of 0.75 / sqrt(2040)).
    To nearest it stays where it was, since a step moves it by 0.1 % and the spacing is 12 to 25 %."""
    n, b2 = 2048, np.float32(0.999)
    g = np.ones(n, dtype=np.float32)
    small = np.where(np.arange(n) % 256 == 0, 1.0, 0.1).astype(np.float32)
    start = orc.scales(np.ones(n, dtype=np.float32), 57344.0)
    v8, s = orc.codes(np.ones(n, dtype=np.float32), start, np.zeros(n, dtype=np.int64), "v"), start
    nearest, s_near = v8.copy(), s.copy()
    quiet = np.arange(n) % 256 != 0
    v0 = float((orc.widen(v8, "v") * np.repeat(s, 256))[1])
    assert abs(v0 - 6 / 7) < 1e-5
    r = np.random.default_rng(2)
    for _ in range(3000):
        step = lambda c, sc: b2 * (orc.widen(c, "v") * np.repeat(sc, 256)) + np.float32(0.001) * small * small  # noqa: E731
        v = step(v8, s)
        s = orc.scales(v, 57344.0)
        v8 = orc.codes(v, s, r.integers(0, 2 ** 21, n), "v")
        v = step(nearest, s_near)
        s_near = orc.scales(v, 57344.0)
        nearest = orc.codes(v, s_near, np.full(n, 2 ** 20), "v")
    got = (orc.widen(v8, "v") * np.repeat(s, 256))[quiet].mean()
    want = 0.01 + (v0 - 0.01) * 0.999 ** 3000
    assert abs(got - want) < 0.06 * want
    assert (orc.widen(nearest, "v") * np.repeat(s_near, 256))[quiet].mean() > 0.5


# ---- CPU: refusals ------------------------------------------------------------------------------------
def _entry(n=1, rows=False, bits=32, lr=1e-3, lr_dev=None, betas=(0.9, 0.999), eps=1e-8, wd=0.0, norm=None, max_norm=1.0, step=512,
           count=None, table=True, **tensor):
    """Calls a step's C entry with addresses that nothing may touch; every such call has to be refused."""
    lib = nv.load()
    words = dict(param=1 << 20, grad=2 << 20, m=3 << 20, v=4 << 20, ms=5 << 20, vs=6 << 20, master=0, numel=512, cols=256,
                 pdt=nv.F32, gdt=nv.F32)
    rows_of = []
    for i in range(n):
        w = {**words, **{k: (x[i] if isinstance(x, (list, tuple)) else x) for k, x in tensor.items()}}
        for k in ("param", "grad", "m", "v", "ms", "vs"):       # tensors of their own, unless the case places them
            if k not in tensor:
                w[k] += i << 24
        rows_of += [w["param"], w["grad"], w["m"], w["v"], w["ms"], w["vs"], w["master"], w["numel"], w["cols"], w["pdt"] | w["gdt"] << 32]
    t = (ctypes.c_int64 * max(1, len(rows_of)))(*rows_of) if table else None
    count = n if count is None else count
    if rows:
        rc = lib.flexsae_adamw_unit_rows_step(t, count, step, lr, lr_dev, *betas, eps, wd, norm, max_norm, None)
    else:
        rc = lib.flexsae_adamw_step(t, count, bits, step, lr, lr_dev, *betas, eps, wd, norm, max_norm, 0, None)
    return rc, lib.flexsae_last_error().decode()


@pytest.mark.parametrize("kw,text", [
    (dict(step=None), "step"), (dict(step=516), "aligned"), (dict(bits=16), "16 bits"),
    (dict(lr=-1.0), "lr"), (dict(lr=math.inf), "lr"), (dict(lr=math.nan), "lr"),
    (dict(betas=(1.0, 0.9)), "betas"), (dict(betas=(0.9, -0.1)), "betas"), (dict(betas=(math.nan, 0.9)), "betas"),
    (dict(eps=0.0), "eps"), (dict(eps=1e-40), "eps"), (dict(eps=math.inf), "eps"), (dict(wd=-1.0), "weight_decay"),
    (dict(norm=64, max_norm=0.0), "max_norm"), (dict(norm=64, max_norm=math.nan), "max_norm"),
    (dict(count=-1), "tensors"), (dict(count=1 << 20), "tensors"), (dict(table=False), "null"),
    (dict(param=0), "null"), (dict(grad=0), "null"), (dict(m=0), "null"), (dict(v=0), "null"),
    (dict(bits=8, ms=0), "scales"), (dict(bits=8, vs=0), "scales"),
    (dict(numel=-1), "numel"), (dict(numel=1 << 39), "numel"), (dict(pdt=7), "dtype"), (dict(pdt=nv.BF16, gdt=nv.F16), "gradient"),
    (dict(pdt=nv.F32, gdt=nv.BF16), "gradient"), (dict(master=7 << 20), "master"),
    (dict(param=(1 << 20) + 2), "aligned"), (dict(pdt=nv.BF16, grad=(2 << 20) + 2), "aligned"), (dict(pdt=nv.BF16, gdt=nv.BF16, param=(1 << 20) + 1), "aligned"),
    (dict(pdt=nv.BF16, master=(7 << 20) + 2), "aligned"), (dict(bits=8, ms=(5 << 20) + 1), "aligned"),
    (dict(grad=1 << 20), "overlap"), (dict(m=(4 << 20) - 4), "overlap"), (dict(bits=8, m=(4 << 20) - 511), "overlap"),
    (dict(bits=8, vs=(5 << 20) + 4), "overlap"), (dict(n=2, param=1 << 20, m=[3 << 20, 7 << 20], v=[4 << 20, 8 << 20]), "twice"),
    (dict(n=2, m=3 << 20), "overlap"), (dict(n=40, v=4 << 20), "overlap"),
    (dict(rows=True, cols=0), "rows"), (dict(rows=True, cols=200), "rows"), (dict(rows=True, numel=16384, cols=16384), "8192"),
])
def test_step_entries_refuse_before_any_launch(kw, text):
    rc, err = _entry(**kw)
    assert rc < 0 and text in err, (rc, err)


@pytest.mark.parametrize("kw", [dict(step=1 << 20), dict(step=(2 << 20) + 8), dict(step=(4 << 20) + 2040), dict(norm=(1 << 20) + 4), dict(lr_dev=3 << 20),
                                dict(norm=512), dict(lr_dev=516), dict(bits=8, step=5 << 20), dict(n=40, norm=(4 << 20) + (30 << 24))])
@pytest.mark.parametrize("rows", [False, True])
def test_a_step_word_norm_or_learning_rate_inside_a_tensor_is_refused(kw, rows):
    """A step reads them while it writes the tensors, and writes the step word while it reads the gradients."""
    if not (rows and "bits" in kw):
        rc, err = _entry(rows=rows, **kw)
        assert rc < 0 and "overlap" in err, (rc, err)


def test_norm_entry_refuses_before_any_launch():
    lib = nv.load()
    size = ctypes.c_size_t()

    def workspace(n, elements):
        assert lib.flexsae_grad_norm_workspace_bytes(n, elements, ctypes.byref(size)) == 0
        return size.value

    assert lib.flexsae_grad_norm_workspace_bytes(-1, 8, ctypes.byref(size)) == -1
    assert lib.flexsae_grad_norm_workspace_bytes(1 << 17, 8, ctypes.byref(size)) == -1
    assert lib.flexsae_grad_norm_workspace_bytes(2, -1, ctypes.byref(size)) == -1
    assert lib.flexsae_grad_norm_workspace_bytes(2, 8, None) == -1
    assert workspace(32, 1 << 18) == 0                            # one cluster, no scratch memory
    large = 1 << 20
    need = workspace(2, large)
    assert need > 0 and workspace(33, 8) > 0 and workspace(32, (1 << 18) + 1) > 0

    def call(grads=(64, 1 << 30), numel=(large, 4), dtypes=(0, 1), n=2, out=512, ws=1024, ws_bytes=need):
        return lib.flexsae_grad_norm((ctypes.c_void_p * 2)(*grads), (ctypes.c_int64 * 2)(*numel), (ctypes.c_int32 * 2)(*dtypes), n, out, ws,
                                     ws_bytes, None), lib.flexsae_last_error().decode()

    for kw, text in ((dict(n=-1), "tensors"), (dict(out=None), "null"), (dict(out=514), "norm_out"), (dict(ws=None), "workspace"),
                     (dict(ws=1028), "aligned"), (dict(ws_bytes=need - 1), "too small"), (dict(dtypes=(0, 5)), "dtype"),
                     (dict(numel=(large, -4)), "numel"), (dict(grads=(64, 0)), "null"), (dict(grads=(66, 128)), "aligned"),
                     (dict(grads=(64, 129)), "aligned")):
        rc, err = call(**kw)
        assert rc < 0 and text in err, (kw, rc, err)
    assert lib.flexsae_grad_norm(None, None, None, 2, 512, 1024, need, None) == -1


def test_norm_of_more_elements_than_its_workspace_counts_on_is_refused():
    """A tensor may be given many times: 256 of 2^36.4 elements (all of a GPU's memory, once) filled three launches' partial sums
    where the workspace holds two.  Lists of up to 2^42 elements in all need one launch for every 256 tensors."""
    lib = nv.load()
    size = ctypes.c_size_t()
    assert lib.flexsae_grad_norm_workspace_bytes(1 << 16, 1 << 42, ctypes.byref(size)) == 0
    need = size.value
    assert lib.flexsae_grad_norm_workspace_bytes(256, (1 << 42) + 1, ctypes.byref(size)) == -1
    n, numel = 256, 90_000_000_000
    rc = lib.flexsae_grad_norm((ctypes.c_void_p * n)(*[1 << 20] * n), (ctypes.c_int64 * n)(*[numel] * n), (ctypes.c_int32 * n)(*[nv.F16] * n), n, 512,
                               1024, need, None)
    assert rc == -1 and "elements" in lib.flexsae_last_error().decode()


def test_python_entries_need_cuda_tensors():
    p, step = torch.zeros(8), torch.zeros((), dtype=torch.int64)
    with pytest.raises(RuntimeError, match="CUDA"):
        optim.adamw_step([p], [p.clone()], [p.clone()], [p.clone()], step, lr=1e-3)
    with pytest.raises(RuntimeError, match="CUDA"):
        optim.grad_norm([p])
    with pytest.raises(ValueError):
        optim.grad_norm([])
    with pytest.raises(ValueError):
        optim.adamw_step([], [], [], [], step, lr=1e-3)
    with pytest.raises(ValueError, match="gradients"):
        optim.adamw_step([p], [], [p], [p], step, lr=1e-3)


def test_optimizer_class_refuses_what_it_cannot_do():
    p, q = torch.nn.Parameter(torch.zeros(4, 8)), torch.nn.Parameter(torch.zeros(8))
    for bad in (dict(state_bits=16), dict(state_bits=8, unit_rows=True), dict(max_norm=0.0), dict(max_norm=-1.0), dict(seed=-1), dict(seed=2 ** 32)):
        with pytest.raises(ValueError):
            optim.AdamW([p], **bad)
    with pytest.raises(ValueError, match="unit rows"):
        optim.AdamW([q], unit_rows=True)
    with pytest.raises(TypeError):
        optim.AdamW([torch.nn.Parameter(torch.zeros(4, dtype=torch.float64))])
    opt = optim.AdamW([p], unit_rows=True)
    with pytest.raises(ValueError):
        opt.add_param_group({"params": [q], "unit_rows": True})
    assert len(opt.param_groups) == 1                              # a refused group is not kept


# ---- CPU: loading states ---------------------------------------------------------------------------------
def theirs_after_a_step(groups, cls=torch.optim.AdamW, **kw):
    """A torch optimizer over ``groups`` (lists of parameters) that has taken one step."""
    opt = cls([{"params": ps} for ps in groups], **{**dict(lr=1e-3), **kw})
    for ps in groups:
        for p in ps:
            p.grad = torch.randn(p.shape, generator=torch.Generator().manual_seed(p.numel())).to(p.dtype)
    opt.step()
    return opt


def test_options_of_a_group_outlive_a_state_that_does_not_know_them():
    """torch.optim.AdamW's groups say nothing of unit rows, master copies, seeds: each group keeps its own."""
    w, b, d = (torch.nn.Parameter(torch.randn(s).to(t)) for s, t in (((6, 8), torch.bfloat16), ((6,), torch.float32), ((6, 8), torch.float32)))
    theirs = theirs_after_a_step([[w], [b], [d]], lr=7e-3)
    ours = optim.AdamW([{"params": [w], "master_weights": True}, {"params": [b]}, {"params": [d], "unit_rows": True, "seed": 3}], lr=1e-3, seed=8)
    ours.load_state_dict(theirs.state_dict())
    got = [(x["lr"], x["unit_rows"], x["master_weights"], x["seed"], x["state_bits"]) for x in ours.param_groups]
    assert got == [(7e-3, False, True, 8, 32), (7e-3, False, False, 8, 32), (7e-3, True, False, 3, 32)]
    assert torch.equal(ours.state[w]["master"], w.detach().float())
    assert "master" not in ours.state[b] and "master" not in ours.state[d]
    # a state of its own says all of it, and is followed
    other = optim.AdamW([{"params": [torch.nn.Parameter(p.detach().clone())]} for p in (w, b, d)], lr=1e-2)
    other.load_state_dict(ours.state_dict())
    assert [(x["lr"], x["unit_rows"], x["master_weights"], x["seed"], x["state_bits"]) for x in other.param_groups] == got


@pytest.mark.parametrize("cls,kw,text", [
    (torch.optim.AdamW, dict(maximize=True), "maximize"), (torch.optim.AdamW, dict(amsgrad=True), "amsgrad"),
    (torch.optim.Adam, dict(weight_decay=0.1), "weight_decay"), (torch.optim.NAdam, {}, "torch.optim.AdamW"),
    (torch.optim.RAdam, {}, "torch.optim.AdamW"), (torch.optim.RAdam, dict(decoupled_weight_decay=True), "torch.optim.AdamW"),
    (torch.optim.SGD, dict(momentum=0.9), "exp_avg"),
])
def test_states_of_other_rules_are_refused_before_anything_changes(cls, kw, text):
    p, q = (torch.nn.Parameter(torch.randn(5, 8)) for _ in range(2))
    ours = optim.AdamW([{"params": [p]}, {"params": [q]}], lr=2e-3)
    ours.load_state_dict(theirs_after_a_step([[p], [q]], lr=2e-3).state_dict())
    kept = {x: dict(ours.state[x]) for x in (p, q)}
    with pytest.raises(ValueError, match=text):
        ours.load_state_dict(theirs_after_a_step([[p], [q]], cls, **kw).state_dict())
    assert all(ours.state[x][name] is value for x in (p, q) for name, value in kept[x].items())
    assert ours.param_groups[0]["lr"] == 2e-3
    # without decay Adam is the same rule
    ours.load_state_dict(theirs_after_a_step([[p], [q]], torch.optim.Adam).state_dict())
    assert ours.param_groups[0]["lr"] == 1e-3


def with_states8(p, seed=0, **kw):
    """An optimizer with made-up 8-bit states of ``p`` (every scale another), and what they stand for."""
    opt = optim.AdamW([p], state_bits=8, **kw)
    state = opt._new_state(p, opt.param_groups[0], torch.tensor(3))
    g = torch.Generator().manual_seed(seed)
    for name, top in (("exp_avg", 0x7F), ("exp_avg_sq", 0x7C)):
        state[name].view(torch.uint8).copy_(torch.randint(1, top, p.shape, generator=g))
        state[name + "_scale"].copy_(1.0 + torch.arange(optim.state8_blocks(p.numel())))
    opt.state[p].update(state)
    return opt


def values8(opt, p, name):
    """What the 8-bit state of ``p`` stands for: its scales go with the elements in memory order."""
    state = opt.state[p]
    order = torch.arange(p.numel()).as_strided(p.shape, p.stride())
    return state[name].float() * state[name + "_scale"][order // 256]


def test_float_moments_are_not_loaded_into_8_bit_states_nor_codes_into_32_bit_ones():
    p = torch.nn.Parameter(torch.randn(5, 8))
    theirs = theirs_after_a_step([[p]])
    ours = optim.AdamW([p], state_bits=8)
    with pytest.raises(TypeError, match="8-bit"):
        ours.load_state_dict(theirs.state_dict())
    assert not ours.state
    eight = with_states8(p).state_dict()
    ours.load_state_dict(eight)
    for name in ("exp_avg", "exp_avg_sq"):
        assert ours.state[p][name].dtype in optim.STATE8_DTYPES and torch.equal(values8(ours, p, name), values8(with_states8(p), p, name))
    for broken in (dict(state_bits=32), dict(params=[0])):              # a group that says otherwise, or that says nothing
        groups = [{k: v for k, v in {**eight["param_groups"][0], **broken}.items() if k != "state_bits" or "params" not in broken}]
        ours = optim.AdamW([p])
        with pytest.raises(TypeError, match="32-bit"):
            ours.load_state_dict({**eight, "param_groups": groups})
        assert not ours.state
    without = {**eight, "state": {0: {k: v for k, v in eight["state"][0].items() if k != "exp_avg_scale"}}}
    with pytest.raises(ValueError, match="exp_avg_scale"):
        optim.AdamW([p], state_bits=8).load_state_dict(without)


@pytest.mark.parametrize("shape", [(64, 40), (4, 512)])
def test_8_bit_states_of_another_layout_are_refused(shape):
    """A scale belongs to 256 elements that lie side by side: in another order its elements are others."""
    plain = torch.nn.Parameter(torch.randn(shape))
    turned = torch.nn.Parameter(torch.randn(shape[::-1]).t())
    for p, q in ((plain, turned), (turned, plain)):
        saved = with_states8(p)
        ours = optim.AdamW([q], state_bits=8)
        with pytest.raises(ValueError, match="layout"):
            ours.load_state_dict(saved.state_dict())
        assert not ours.state
        ours = optim.AdamW([torch.nn.Parameter(p.detach().clone())], state_bits=8)
        ours.load_state_dict(saved.state_dict())
        for name in ("exp_avg", "exp_avg_sq"):
            assert torch.equal(values8(ours, ours.param_groups[0]["params"][0], name), values8(saved, p, name))
    wide = optim.AdamW([turned])                                       # 32-bit states go by their elements
    wide.load_state_dict(theirs_after_a_step([[plain]]).state_dict())
    assert wide.state[turned]["exp_avg"].stride() == turned.stride()


def test_states_of_other_shapes_are_refused_and_further_entries_are_left_alone():
    p, q = torch.nn.Parameter(torch.randn(8)), torch.nn.Parameter(torch.randn(4, 8))
    for saved, kw in ((theirs_after_a_step([[p]]), {}), (with_states8(p), dict(state_bits=8))):
        ours = optim.AdamW([q], **kw)
        with pytest.raises(ValueError, match="shape"):
            ours.load_state_dict(saved.state_dict())
        assert not ours.state
    w = torch.nn.Parameter(torch.randn(4, 8).bfloat16())
    ours = optim.AdamW([w], master_weights=True)
    ours.state[w].update(ours._new_state(w, ours.param_groups[0], torch.tensor(1)))
    state = ours.state_dict()
    with pytest.raises(ValueError, match="shape"):
        ours.load_state_dict({**state, "state": {0: {**state["state"][0], "master": torch.zeros(8)}}})
    eight = with_states8(q).state_dict()
    with pytest.raises(ValueError, match="exp_avg_scale"):
        optim.AdamW([q], state_bits=8).load_state_dict({**eight, "state": {0: {**eight["state"][0], "exp_avg_scale": torch.zeros(2)}}})
    # what a program keeps beside the states comes as the base class has it
    ours.load_state_dict({**state, "state": {0: {**state["state"][0], "seen": 5, "age": torch.arange(3)}}})
    assert ours.state[w]["seen"] == 5 and ours.state[w]["age"].shape == (3,)


def test_hooks_around_loading_see_and_set_the_states():
    """A hook before may replace the state, one after sees the restored states and may change them."""
    p, q = torch.nn.Parameter(torch.randn(5, 8).bfloat16()), torch.nn.Parameter(torch.randn(8))
    theirs = theirs_after_a_step([[p], [q]])
    ours = optim.AdamW([{"params": [p], "master_weights": True}, {"params": [q]}])
    seen = []

    def before(opt, state):
        assert opt is ours
        seven = {**state["state"][0], "exp_avg": torch.full((5, 8), 7.0)}
        return {"state": {**state["state"], 0: seven}, "param_groups": [{**g, "lr": 0.5} for g in state["param_groups"]]}

    def after(opt):
        seen.append({name: x.dtype for name, x in opt.state[p].items()})
        opt.state[q]["exp_avg"] = torch.full((8,), 9.0)

    handles = [ours.register_load_state_dict_pre_hook(before), ours.register_load_state_dict_post_hook(after)]
    ours.load_state_dict(theirs.state_dict())
    assert seen == [{"step": torch.int64, "exp_avg": torch.float32, "exp_avg_sq": torch.float32, "master": torch.float32}]
    assert bool((ours.state[p]["exp_avg"] == 7).all()) and bool((ours.state[q]["exp_avg"] == 9).all())
    assert [(g["lr"], g["master_weights"]) for g in ours.param_groups] == [(0.5, True), (0.5, False)]
    for h in handles:
        h.remove()
    ours.load_state_dict(theirs.state_dict())                          # and nothing of a load stays behind
    assert len(seen) == 1 and ours.param_groups[0]["lr"] == 1e-3
    ours.register_load_state_dict_pre_hook(lambda opt, state: {**state, "param_groups": [{**g, "maximize": True} for g in state["param_groups"]]})
    with pytest.raises(ValueError, match="maximize"):
        ours.load_state_dict(theirs.state_dict())
    assert ours.param_groups[0]["lr"] == 1e-3 and not ours.param_groups[0].get("maximize")


def test_master_copies_are_not_loaded_beside_32_bit_parameters():
    """A state of 16-bit weights with master copies, loaded into a model that is held in 32 bits: a step refuses masters there."""
    w = torch.nn.Parameter(torch.randn(4, 8).bfloat16())
    sixteen = optim.AdamW([w], master_weights=True)
    sixteen.state[w].update(sixteen._new_state(w, sixteen.param_groups[0], torch.tensor(1)))
    q = torch.nn.Parameter(w.detach().float())
    ours = optim.AdamW([q])
    ours.load_state_dict(sixteen.state_dict())
    assert sorted(ours.state[q]) == ["exp_avg", "exp_avg_sq", "step"]


@pytest.mark.parametrize("theirs,ours,text", [
    (dict(state_bits=8), dict(unit_rows=True), "unit_rows"), (dict(state_bits=16), {}, "state_bits"), (dict(seed=-1), {}, "seed"),
    (dict(unit_rows=True), dict(shape=(8,)), "unit rows"),
])
def test_options_that_do_not_go_together_are_refused_at_load_too(theirs, ours, text):
    p = torch.nn.Parameter(torch.randn(ours.get("shape", (4, 8))))
    opt = optim.AdamW([p], lr=2e-3, **{k: v for k, v in ours.items() if k != "shape"})
    with pytest.raises(ValueError, match=text):
        opt.load_state_dict({"state": {}, "param_groups": [{"params": [0], "lr": 1e-3, **theirs}]})
    assert opt.param_groups[0]["lr"] == 2e-3 and opt.param_groups[0]["state_bits"] == 32


# ---- CPU: step counts ------------------------------------------------------------------------------------
def let_take_part(ps, active):
    for k, p in enumerate(ps):
        p.grad = torch.ones_like(p) if k in active else None


def cohorts_of(opt, ps):
    """The positions of the parameters that step together, with their counts moved as the step would."""
    where = {id(p): k for k, p in enumerate(ps)}
    cohorts = opt._cohorts(opt.param_groups[0])
    for c in cohorts:
        opt.state[c[0]]["step"].add_(1)
    return [[where[id(p)] for p in c] for c in cohorts]


def test_parameters_that_sit_out_together_go_on_together():
    ps = [torch.nn.Parameter(torch.ones(3)) for _ in range(5)]
    opt = optim.AdamW(ps)
    for active, want in (((0, 1, 2, 3, 4), [[0, 1, 2, 3, 4]]), ((0,), [[0]]), ((0, 1, 2, 3, 4), [[0], [1, 2, 3, 4]]), ((0, 1, 2), [[0], [1, 2]]),
                         ((0, 1, 2, 3, 4), [[0], [1, 2], [3, 4]])):
        let_take_part(ps, active)
        assert cohorts_of(opt, ps) == want
    assert [int(opt.state[p]["step"]) for p in ps] == [5, 4, 4, 3, 3]


def test_cohorts_of_a_group_round_independently(monkeypatch):
    """Parameters that stand at the same count, but step in different calls, are both first in their lists: the random bits of
    those calls need different seeds, and the bits of a parameter that is first in its group those of the group's seed."""
    calls = []
    monkeypatch.setattr(optim, "adamw8_step", lambda ps, *a, seed, **kw: calls.append((tuple(id(p) for p in ps), seed)) or a[-1].add_(1))
    ps = [torch.nn.Parameter(torch.ones(3)) for _ in range(4)]
    opt = optim.AdamW(ps, state_bits=8, seed=2 ** 32 - 1)
    first, where = 2 ** 32 - 1, [id(p) for p in ps]
    let_take_part(ps, (0, 1, 2, 3))
    opt.step()
    assert calls == [(tuple(where), first)]
    for active in ((1, 2, 3), (0, 2, 3), (0, 1, 3), (0, 1, 2)):
        let_take_part(ps, active)
        opt.step()
    assert len({int(opt.state[p]["step"]) for p in ps}) == 1             # each sat out once: apart, at the same count
    calls.clear()
    let_take_part(ps, (0, 1, 2, 3))
    opt.step()
    assert sorted(c[0] for c in calls) == sorted((i,) for i in where)
    seeds = {c[0][0]: c[1] for c in calls}
    assert len(set(seeds.values())) == 4 and seeds[where[0]] == first and all(0 <= x < 2 ** 32 for x in seeds.values())
    calls.clear()
    opt.step()
    assert {c[0][0]: c[1] for c in calls} == seeds                     # a parameter keeps its own


# ---- GPU: helpers ---------------------------------------------------------------------------------------
def f64(t):
    return t.detach().double().cpu().numpy()


def steps_in(name):
    return torch.tensor(name, dtype=torch.int64, device="cuda")


def make(shape, dtype, seed, master=False, grad_dtype=None, offset=0, spread=True):
    """(p, g, m, v, master) on the GPU, optionally ``offset`` elements into their storage; some gradients are zero."""
    g = torch.Generator().manual_seed(seed)
    n = math.prod(shape)

    def place(x, dt):
        store = torch.zeros(n + offset, dtype=dt, device="cuda")
        return store[offset:].view(shape).copy_(x)

    p = torch.randn(shape, generator=g)
    grad = torch.randn(shape, generator=g) * 1e-2
    if spread:
        grad = grad * 10.0 ** (torch.rand(shape, generator=g) * 3 - 2)
    grad[torch.rand(shape, generator=g) < 0.1] = 0
    m, v = torch.randn(shape, generator=g) * 3e-3, torch.randn(shape, generator=g).square() * 1e-5
    return (place(p, dtype), place(grad, grad_dtype or dtype), place(m, torch.float32), place(v, torch.float32),
            place(p, torch.float32) if master else None)


def bounds(before, after, t, lr, betas, eps, clip):
    """Allowed errors of (p, m, v), see the head of this file; ``after`` is the oracle's answer."""
    p, g, m, v = (np.abs(x) for x in before)
    g = g * clip
    em = U * (3 * betas[0] * m + 8 * (1 - betas[0]) * g)
    ev = U * (3 * betas[1] * v + 13 * (1 - betas[1]) * g * g)
    denom = np.sqrt(after[2]) / math.sqrt(1 - betas[1] ** t) + eps
    rate = lr / (1 - betas[0] ** t)
    relative_v = np.divide(ev, after[2], out=np.zeros_like(ev), where=after[2] > 0) / 2
    step = rate * np.abs(after[1]) / denom
    return 4 * U * p + (24 * U + relative_v) * step + rate * em / denom, em + 2.0 ** -149, ev + 2.0 ** -148


def close(got, want, bound, what):
    bad = ~(np.abs(f64(got) - want) <= bound)
    assert not bad.any(), (what, int(bad.sum()), np.abs(f64(got) - want)[bad][:4], np.broadcast_to(bound, bad.shape)[bad][:4])


def check_params(p, master, want, bound, dtype):
    half, tiny = HALF[dtype]
    close(p, want, bound + half * np.abs(want) + half * bound + tiny, "param")
    if master is not None:
        close(master, want, bound, "master")
        assert torch.equal(p, master.to(dtype))                     # the parameter is its copy, rounded


# ---- GPU: gradient norm ------------------------------------------------------------------------------------
# 32-bit sums of eight squares (8 u), then 64 bits; the root halves that and the result is rounded: 5 u
NORM_TOL = 5 * U


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,offset", [(1, 0), (7, 0), (255, 1), (256, 0), (257, 3), (8191, 0), (8192, 0), (8193, 1), (100003, 0), (1 << 18, 0), ((1 << 18) + 1, 0), (20_000_001, 0)])
def test_norm_of_one_tensor(dtype, n, offset):
    x = torch.randn(n + offset, generator=torch.Generator().manual_seed(n)).to(dtype).cuda()[offset:]
    want = float(x.double().square().sum().sqrt())
    got = optim.grad_norm([x])
    assert got.dtype == torch.float32 and got.shape == () and abs(float(got) - want) <= NORM_TOL * want
    assert torch.equal(got, optim.grad_norm([x]))


@gpu
@pytest.mark.parametrize("count", [2, 16, 17, 30, 31, 256, 257, 600])
def test_norm_of_many_mixed_tensors(count):
    g = torch.Generator().manual_seed(count)
    dtypes = [torch.float32, torch.bfloat16, torch.float16]
    xs = [torch.randn((i * 37) % 501, generator=g).to(dtypes[i % 3]).cuda() for i in range(count)]
    xs.append(torch.randn(50, 60, generator=g).cuda().t())                              # dense, another order
    xs.append(torch.randn(50, 60, generator=g).cuda()[:, ::2])                         # with gaps
    want = math.sqrt(sum(float(x.double().square().sum()) for x in xs))
    assert abs(float(optim.grad_norm(xs)) - want) <= NORM_TOL * want


@gpu
def test_norm_of_extreme_values():
    big = torch.full((1000,), 1e30, device="cuda")
    assert abs(float(optim.grad_norm([big])) - float(big[0]) * math.sqrt(1000)) <= NORM_TOL * 1e30 * 32
    small = torch.full((1000,), 1e-30, device="cuda")
    small[::3] = 0
    assert abs(float(optim.grad_norm([small])) - float(small.double().square().sum().sqrt())) <= NORM_TOL * 1e-28
    assert float(optim.grad_norm([torch.zeros(5000, device="cuda")])) == 0
    assert float(optim.grad_norm([torch.empty(0, device="cuda")])) == 0
    for bad in (math.inf, -math.inf):
        big[17] = bad
        assert float(optim.grad_norm([small, big])) == math.inf
    big[18] = math.nan
    assert math.isnan(float(optim.grad_norm([small, big])))


# ---- GPU: AdamW, 32-bit states ------------------------------------------------------------------------
KINDS = [(torch.float32, torch.float32, False)] + [(d, g, m) for d in (torch.bfloat16, torch.float16)
                                                   for g in (d, torch.float32) for m in (False, True)]
SHAPES = [(1,), (3,), (255,), (256,), (257,), (2047,), (2049,), (1, 4096), (61, 77), (1000, 129)]


@gpu
@pytest.mark.parametrize("dtype,grad_dtype,master", KINDS)
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("t", [1, 1000])
def test_adamw_against_the_oracle(dtype, grad_dtype, master, offset, t):
    sets = [make(s, dtype, 100 * k + offset, master, grad_dtype, offset) for k, s in enumerate(SHAPES)]
    if t == 1:
        for x in sets:
            x[2].zero_(), x[3].zero_()
    before = [[f64(x[4] if master else x[0]), f64(x[1]), f64(x[2]), f64(x[3])] for x in sets]
    kw = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-6, weight_decay=0.1)
    step = steps_in(t - 1)
    optim.adamw_step(*[[x[k] for x in sets] for k in range(4)], step, masters=[x[4] for x in sets] if master else None, **kw)
    assert int(step) == t
    for x, b in zip(sets, before):
        want = orc.adamw(*b, t, 3e-3, (0.9, 0.99), 1e-6, 0.1)
        ep, em, ev = bounds(b, want, t, 3e-3, (0.9, 0.99), 1e-6, 1.0)
        check_params(x[0], x[4], want[0], ep, dtype)
        close(x[2], want[1], em, "m")
        close(x[3], want[2], ev, "v")


@gpu
def test_adamw_on_many_tensors_of_all_kinds_with_empty_ones():
    """Over 256 tensors of one kind, every other kind beside them, empty tensors among them: every element is updated
    once and the count moves by one."""
    sets, masters = [], []
    for i in range(330):
        dtype, grad_dtype, master = KINDS[0] if i < 300 else KINDS[i % len(KINDS)]
        x = make(((i * 131) % 700,), dtype, i, master, grad_dtype)
        sets.append(x)
        masters.append(x[4])
    before = [[f64(x[4] if x[4] is not None else x[0]), f64(x[1]), f64(x[2]), f64(x[3])] for x in sets]
    step = steps_in(4)
    optim.adamw_step(*[[x[k] for x in sets] for k in range(4)], step, lr=1e-3, masters=masters)
    assert int(step) == 5
    for x, b in zip(sets, before):
        want = orc.adamw(*b, 5, 1e-3)
        ep, em, ev = bounds(b, want, 5, 1e-3, (0.9, 0.999), 1e-8, 1.0)
        check_params(x[0], x[4], want[0], ep, x[0].dtype)
        close(x[2], want[1], em, "m")
        close(x[3], want[2], ev, "v")


@gpu
@pytest.mark.parametrize("dtype,grad_dtype,master", KINDS)
def test_adamw_long_lists_of_every_kind(dtype, grad_dtype, master):
    sets = [make((1024 * (k % 3) + 40 * k + 1,), dtype, 300 + k, master, grad_dtype) for k in range(40)]
    before = [[f64(x[4] if master else x[0]), f64(x[1]), f64(x[2]), f64(x[3])] for x in sets]
    optim.adamw_step(*[[x[k] for x in sets] for k in range(4)], steps_in(6), lr=1e-3, masters=[x[4] for x in sets])
    for x, b in zip(sets, before):
        want = orc.adamw(*b, 7, 1e-3)
        ep, em, ev = bounds(b, want, 7, 1e-3, (0.9, 0.999), 1e-8, 1.0)
        check_params(x[0], x[4], want[0], ep, dtype)
        close(x[2], want[1], em, "m"), close(x[3], want[2], ev, "v")


@gpu
def test_only_empty_tensors_still_count_the_step():
    e, step = [torch.empty(0, device="cuda") for _ in range(4)], steps_in(7)
    optim.adamw_step(*[[x] for x in e], step, lr=1e-3)
    assert int(step) == 8
    e = [torch.empty(0, 8, device="cuda") for _ in range(4)]
    optim.adamw_unit_rows_step(*[[x] for x in e], step, lr=1e-3)
    assert int(step) == 9


@gpu
@pytest.mark.parametrize("max_norm", [0.25, 1e9])
def test_clipping_uses_the_norm_on_the_device(max_norm):
    x = make((300, 70), torch.float32, 5)
    b = [f64(t) for t in x[:4]]
    norm = optim.grad_norm([x[1]])
    step = steps_in(9)
    optim.adamw_step(*[[t] for t in x[:4]], step, lr=1e-2, norm=norm, max_norm=max_norm)
    clip = orc.clip_factor(float(norm), max_norm)
    assert clip < 1 if max_norm < 1 else clip == 1
    want = orc.adamw(*b, 10, 1e-2, clip=clip)
    ep, em, ev = bounds(b, want, 10, 1e-2, (0.9, 0.999), 1e-8, clip)
    close(x[0], want[0], ep, "param"), close(x[2], want[1], em, "m"), close(x[3], want[2], ev, "v")


@gpu
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("entry", ["adamw", "adamw8", "rows"])
def test_a_norm_that_is_not_finite_leaves_everything(bad, entry):
    x, step, norm = make((40, 64), torch.bfloat16, 6, master=True), steps_in(3), torch.tensor(bad, device="cuda")
    m, v = x[2], x[3]
    if entry == "adamw8":
        m, v = (torch.randint(0, 100, (40, 64), dtype=torch.uint8, device="cuda").view(d) for d in optim.STATE8_DTYPES)
    scales = [torch.rand(10, device="cuda") for _ in range(2)]
    state = [x[0], x[4], m.view(torch.uint8), v.view(torch.uint8), *scales, step]
    kept = [t.clone() for t in state]
    kw = dict(lr=1e-3, norm=norm, masters=[x[4]])
    if entry == "adamw8":
        optim.adamw8_step([x[0]], [x[1]], [m], [scales[0]], [v], [scales[1]], step, max_norm=1.0, **kw)
    else:
        (optim.adamw_step if entry == "adamw" else optim.adamw_unit_rows_step)([x[0]], [x[1]], [m], [v], step, **kw)
    for a, b in zip(state, kept):
        assert torch.equal(a, b)


@gpu
def test_nonfinite_gradients_without_a_norm_stay_with_their_elements():
    x = make((1000,), torch.float32, 7)
    y = [t.clone() for t in x[:4]]
    x[1][123], x[1][700] = math.nan, math.inf
    optim.adamw_step(*[[t] for t in x[:4]], steps_in(0), lr=1e-3)
    optim.adamw_step(*[[t] for t in y], steps_in(0), lr=1e-3)
    keep = torch.ones(1000, dtype=torch.bool, device="cuda")
    keep[[123, 700]] = False
    for a, b in zip((x[0], x[2], x[3]), (y[0], y[2], y[3])):
        assert torch.equal(a[keep], b[keep]) and not torch.isfinite(a[~keep]).any()


@gpu
def test_layouts_transposed_parameters_and_foreign_gradients():
    """A transposed parameter with states like it; a gradient in another order is brought into it."""
    p, g, m, v, _ = make((48, 80), torch.float32, 8)
    b = [f64(t) for t in (p, g, m, v)]
    pt, mt, vt = (torch.empty(80, 48, device="cuda").t().copy_(t) for t in (p, m, v))
    step = steps_in(0)
    optim.adamw_step([pt], [g], [mt], [vt], step, lr=1e-3)
    want = orc.adamw(*b, 1, 1e-3)
    ep, em, ev = bounds(b, want, 1, 1e-3, (0.9, 0.999), 1e-8, 1.0)
    close(pt, want[0], ep, "param"), close(mt, want[1], em, "m"), close(vt, want[2], ev, "v")


@gpu
def test_lazily_negated_views():
    """A view whose memory holds the negated values (torch keeps such for parts of conjugates): a gradient is read as what it stands for,
    what a step writes or reads as a word is refused."""
    x = make((48, 80), torch.float32, 8)
    y, step = [t.clone() for t in x[:4]], steps_in(0)
    negated = torch._neg_view(-x[1])
    assert torch.equal(negated, x[1]) and negated.is_neg()
    optim.adamw_step([x[0]], [negated], [x[2]], [x[3]], step, lr=1e-3)
    optim.adamw_step(*[[t] for t in y], steps_in(0), lr=1e-3)
    assert torch.equal(x[0], y[0]) and torch.equal(x[2], y[2])
    norm = torch.ones((), device="cuda")
    for k, kw in ((0, {}), (2, {}), (3, {}), (None, dict(norm=torch._neg_view(norm))), (None, dict(lr=torch._neg_view(norm)))):
        args = [[torch._neg_view(t) if i == k else t] for i, t in enumerate(y)]
        with pytest.raises(ValueError, match="negated"):
            optim.adamw_step(*args, step, **{**dict(lr=1e-3), **kw})


@gpu
def test_python_refusals_on_cuda_tensors():
    p, g, m, v, _ = make((16, 32), torch.bfloat16, 9)
    step = steps_in(0)

    def call(p=p, g=g, m=m, v=v, step=step, **kw):
        optim.adamw_step([p], [g], [m], [v], step, **{**dict(lr=1e-3), **kw})

    for err, kw in (
            (TypeError, dict(p=p.double(), g=g.double())), (TypeError, dict(g=g.half())), (TypeError, dict(g=g.to_sparse())),
            (TypeError, dict(m=m.bfloat16())), (TypeError, dict(step=step.int())), (TypeError, dict(norm=torch.zeros((), device="cuda", dtype=torch.float64))),
            (ValueError, dict(g=g[:8])), (ValueError, dict(m=m[:8])), (ValueError, dict(m=m.t().contiguous().t())),
            (ValueError, dict(p=torch.zeros(16, 64, device="cuda")[:, ::2], g=g.float())), (ValueError, dict(step=torch.zeros(2, dtype=torch.int64, device="cuda"))),
            (ValueError, dict(lr=-1.0)), (ValueError, dict(betas=(0.9, 1.0))), (ValueError, dict(eps=0.0)), (ValueError, dict(weight_decay=math.nan)),
            (ValueError, dict(max_norm=1.0)), (ValueError, dict(norm=torch.zeros((), device="cuda"), max_norm=0.0)),
            (ValueError, dict(p=p.float(), g=g.float(), masters=[m.clone()])), (ValueError, dict(masters=[])), (RuntimeError, dict(m=m.cpu())),
            (RuntimeError, dict(g=g.cpu())), (RuntimeError, dict(step=step.cpu())), (nv.FlexSaeNativeError, dict(v=m))):
        kept = [t.clone() for t in (p, m, v, step)]
        with pytest.raises(err):
            call(**kw)
        assert all(torch.equal(a, b) for a, b in zip((p, m, v, step), kept))
    with pytest.raises(nv.FlexSaeNativeError, match="twice"):
        optim.adamw_step([p, p], [g, g], [m, m.clone()], [v, v.clone()], step, lr=1e-3)
    with pytest.raises(ValueError):
        optim.adamw_unit_rows_step([p.t()], [g.t()], [m.t()], [v.t()], step, lr=1e-3)
    with pytest.raises(ValueError):
        optim.adamw_unit_rows_step([p[0]], [g[0]], [m[0]], [v[0]], step, lr=1e-3)
    with pytest.raises(ValueError, match="seed"):
        optim.adamw8_step([p], [g], [m.to(torch.float8_e4m3fn)], [torch.zeros(2, device="cuda")], [v.to(torch.float8_e5m2)],
                          [torch.zeros(2, device="cuda")], step, lr=1e-3, seed=-1)
    with pytest.raises(ValueError, match="scales"):
        optim.adamw8_step([p], [g], [m.to(torch.float8_e4m3fn)], [torch.zeros(3, device="cuda")], [v.to(torch.float8_e5m2)],
                          [torch.zeros(2, device="cuda")], step, lr=1e-3)


# ---- GPU: 8-bit states ----------------------------------------------------------------------------------
def make8(shape, dtype, seed, master=False, offset=0):
    p, g, m, v, w = make(shape, dtype, seed, master, offset=offset)
    n = p.numel()
    state = []
    for x, kind, largest, dt in ((m, "m", 448.0, torch.float8_e4m3fn), (v, "v", 57344.0, torch.float8_e5m2)):
        flat = x.reshape(-1).cpu().numpy()
        s = orc.scales(flat, largest)
        c = orc.codes(flat, s, np.full(n, 1 << 19), kind)
        store = torch.zeros(n + offset, dtype=torch.uint8, device="cuda")
        store[offset:] = torch.from_numpy(c)
        state += [store[offset:].view(dt).view(shape), torch.from_numpy(s).cuda()]
    return [p, g, *state, w]


def bytes_of(t):
    return t.view(torch.uint8).reshape(-1).cpu().numpy()


@gpu
@pytest.mark.parametrize("dtype,master", [(torch.float32, False), (torch.bfloat16, False), (torch.bfloat16, True), (torch.float16, True)])
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("clipped", [False, True])
def test_adamw8_states_are_the_oracles_bits(dtype, master, offset, clipped):
    """Moments, scales and codes bit for bit as the definition in 32-bit arithmetic gives them; the parameter within
    the bounds of its formula, from the moments before their rounding.  Three steps in a row."""
    sets = [make8(s, dtype, 10 * k, master, offset) for k, s in enumerate(SHAPES)]
    step = steps_in(40)
    norm = torch.tensor(3.0, device="cuda") if clipped else None
    f = np.float32
    clip = min(f(1) / (f(3.0) + f(1e-6)) * f(0.7), f(1)) if clipped else f(1)
    for k in range(3):
        before = [[f64(x[6] if master else x[0]), x[1].float().cpu().numpy().reshape(-1), bytes_of(x[2]), x[3].cpu().numpy(), bytes_of(x[4]),
                   x[5].cpu().numpy()] for x in sets]
        optim.adamw8_step(*[[x[j] for x in sets] for j in range(6)], step, lr=2e-3, eps=1e-6, masters=[x[6] for x in sets] if master else None,
                          norm=norm, max_norm=0.7 if clipped else None, seed=77)
        assert int(step) == 41 + k
        for i, (x, b) in enumerate(zip(sets, before)):
            m, v, m8, ms, v8, vs = orc.adamw8_states(*b[1:], 41 + k, 77, i, clip=clip)
            assert np.array_equal(x[3].cpu().numpy(), ms) and np.array_equal(x[5].cpu().numpy(), vs)
            assert np.array_equal(bytes_of(x[2]), m8) and np.array_equal(bytes_of(x[4]), v8)
            shape = tuple(x[0].shape)
            m, v = m.reshape(shape).astype(np.float64), v.reshape(shape).astype(np.float64)
            t, p = 41 + k, b[0].reshape(shape)
            rate, denom = 2e-3 / (1 - 0.9 ** t), np.sqrt(v) / math.sqrt(1 - 0.999 ** t) + 1e-6
            want = p * (1 - 2e-3 * 0.01) - rate * m / denom
            check_params(x[0], x[6], want, 4 * U * np.abs(p) + 32 * U * rate * np.abs(m) / denom, dtype)


@gpu
@pytest.mark.parametrize("dtype,grad_dtype,master", KINDS)
@pytest.mark.parametrize("count", [2, 40])
def test_adamw8_every_compiled_kernel_rounds_alike(dtype, grad_dtype, master, count):
    """The kernels are compiled for every combination of types and for short and long lists: each of them bit for bit."""
    sets = [make8((4096 + 77,), dtype, 90 + k, master) for k in range(count)]
    for x in sets:
        x[1] = x[1].to(grad_dtype)
    before = [[x[1].float().cpu().numpy(), bytes_of(x[2]), x[3].cpu().numpy(), bytes_of(x[4]), x[5].cpu().numpy()] for x in sets]
    optim.adamw8_step(*[[x[j] for x in sets] for j in range(6)], steps_in(6), lr=2e-3, masters=[x[6] for x in sets], seed=2 ** 32 - 1)
    for i, (x, b) in enumerate(zip(sets, before)):
        _, _, m8, ms, v8, vs = orc.adamw8_states(*b, 7, 2 ** 32 - 1, i)
        assert np.array_equal(x[3].cpu().numpy(), ms) and np.array_equal(x[5].cpu().numpy(), vs)
        assert np.array_equal(bytes_of(x[2]), m8) and np.array_equal(bytes_of(x[4]), v8)


@gpu
def test_adamw8_from_zero_states_and_idle_blocks():
    """First step from nothing; a block without any gradient keeps scales of zero and codes that widen to zero."""
    p = torch.randn(1024, device="cuda")
    g = torch.randn(1024, device="cuda")
    g[256:512] = 0
    p0 = p.clone()
    m, v = torch.zeros(1024, dtype=torch.float8_e4m3fn, device="cuda"), torch.zeros(1024, dtype=torch.float8_e5m2, device="cuda")
    sm, sv, step = torch.zeros(4, device="cuda"), torch.zeros(4, device="cuda"), steps_in(0)
    optim.adamw8_step([p], [g], [m], [sm], [v], [sv], step, lr=1e-3, weight_decay=0.0)
    assert torch.equal(p[256:512], p0[256:512]) and float(sm[1]) == 0 and float(sv[1]) == 0
    sure = g.abs() > 1e-4                                              # eps = 1e-8 takes 1e-4 of the step at most
    sure[256:512] = False
    assert torch.allclose((p0 - p)[sure], 1e-3 * torch.sign(g[sure]), rtol=2e-3, atol=0)
    widened = m.float() * sm.repeat_interleave(256)
    assert bool(((widened - 0.1 * g).abs() <= 0.125 * (0.1 * g).abs() + sm.repeat_interleave(256) * 2.0 ** -9 + 1e-9).all())


@gpu
def test_adamw8_nonfinite_values_stay_with_their_elements():
    sets = [make8((768,), torch.float32, 11) for _ in range(2)]
    sets[0][1][300], sets[0][1][301] = math.nan, math.inf
    before = [sets[0][1].cpu().numpy(), bytes_of(sets[0][2]), sets[0][3].cpu().numpy(), bytes_of(sets[0][4]), sets[0][5].cpu().numpy()]
    for x in sets:
        optim.adamw8_step(*[[x[j]] for j in range(6)], steps_in(0), lr=1e-3, seed=3)
    _, _, m8, ms, v8, vs = orc.adamw8_states(*before, 1, 3, 0)
    x = sets[0]
    assert np.array_equal(bytes_of(x[2]), m8) and np.array_equal(bytes_of(x[4]), v8)
    assert np.array_equal(x[3].cpu().numpy(), ms) and np.array_equal(x[5].cpu().numpy(), vs)
    keep = torch.ones(768, dtype=torch.bool, device="cuda")
    keep[[300, 301]] = False
    assert torch.equal(x[0][keep], sets[1][0][keep]) and not torch.isfinite(x[0][~keep]).any()
    assert torch.isnan(x[2].float()[[300, 301]]).all() and torch.isnan(x[4].float()[300]) and float(x[4].float()[301]) == math.inf


@gpu
@pytest.mark.parametrize("alone", [False, True])
def test_adamw8_second_moment_that_overflows_stays_infinite(alone):
    """As with 32-bit states: the element's parameter stands still from then on and nothing becomes a NaN."""
    x = make8((512,), torch.float32, 13)
    for k in (2, 4):
        x[k].view(torch.uint8).zero_()
        x[k + 1].zero_()
    x[1].copy_(torch.randn(512, generator=torch.Generator().manual_seed(1)) * (0 if alone else 1e-3))
    x[1][300] = 1e30
    kept, step = x[0].clone(), steps_in(0)
    for t in range(3):
        before = [x[1].cpu().numpy(), bytes_of(x[2]), x[3].cpu().numpy(), bytes_of(x[4]), x[5].cpu().numpy()]
        optim.adamw8_step(*[[x[j]] for j in range(6)], step, lr=1e-3, weight_decay=0.0, seed=3)
        _, _, m8, ms, v8, vs = orc.adamw8_states(*before, t + 1, 3, 0)
        assert np.array_equal(bytes_of(x[2]), m8) and np.array_equal(bytes_of(x[4]), v8)
        assert np.array_equal(x[3].cpu().numpy(), ms) and np.array_equal(x[5].cpu().numpy(), vs)
        assert bytes_of(x[4])[300] == 0x7C and torch.isfinite(x[0]).all() and float(x[0][300]) == float(kept[300])
        x[1][300] = 0


@gpu
@pytest.mark.parametrize("scale", [1e-22, 1e15])
def test_adamw8_extreme_gradients(scale):
    """Squares near the ends of the 32-bit range: tiny blocks fall to a scale of zero, large ones stay finite."""
    x = make8((512,), torch.float32, 12)
    x[1].copy_(torch.randn(512, generator=torch.Generator().manual_seed(1)) * scale)
    for k in (2, 4):
        x[k].view(torch.uint8).zero_()
        x[k + 1].zero_()
    before = [x[1].cpu().numpy(), bytes_of(x[2]), x[3].cpu().numpy(), bytes_of(x[4]), x[5].cpu().numpy()]
    optim.adamw8_step(*[[x[j]] for j in range(6)], steps_in(0), lr=1e-3, seed=5)
    _, _, m8, ms, v8, vs = orc.adamw8_states(*before, 1, 5, 0)
    assert np.array_equal(bytes_of(x[2]), m8) and np.array_equal(bytes_of(x[4]), v8)
    assert np.array_equal(x[3].cpu().numpy(), ms) and np.array_equal(x[5].cpu().numpy(), vs)
    assert torch.isfinite(x[0]).all()


@gpu
@pytest.mark.parametrize("eps", [1e-15, 1e-30])
@pytest.mark.parametrize("entry", ["adamw", "adamw8", "rows"])
def test_an_eps_beside_which_tiny_roots_count(eps, entry):
    """Gradients of 1e-17 and below, whose squares are subnormal or zero in 32 bits, with an eps of their size or less.
    A square rounded to a multiple of 2^-149 is off by 2^-150, the rounded product (1 - b2) g^2 by as much again; the root of
    v is then off by at most sqrt(2^-148), which the bound takes beside the usual ones."""
    x = make8((3, 256), torch.float32, 31) if entry == "adamw8" else make((3, 256), torch.float32, 31)
    w = x[0]
    w.copy_(torch.nn.functional.normalize(w, dim=1))
    g = torch.Generator().manual_seed(2)
    x[1].copy_(torch.randn(3, 256, generator=g) * torch.tensor([1e-14, 1e-17, 1e-19])[:, None])
    states = (x[2], x[4]) if entry == "adamw8" else (x[2], x[3])
    for t in states:
        t.view(torch.uint8).zero_()
    if entry == "adamw8":
        x[3].zero_(), x[5].zero_()
    b, grad = f64(w), f64(x[1])
    kw = dict(lr=1e-3, betas=(0.9, 0.99), eps=eps, weight_decay=0.0)
    if entry == "adamw8":
        optim.adamw8_step(*[[t] for t in x[:6]], steps_in(0), **kw)
    else:
        (optim.adamw_step if entry == "adamw" else optim.adamw_unit_rows_step)(*[[t] for t in x[:4]], steps_in(0), **kw)
    if entry == "rows":                                  # the first row's squares are ordinary numbers: the usual bounds
        want = orc.adamw(b, grad, 0 * b, 0 * b, 1, 1e-3, (0.9, 0.99), eps, 0.0, unit_rows=True)
        ep, em, ev = rows_bounds((b, grad, 0 * b, 0 * b), want, 1, 1e-3, 1.0, (0.9, 0.99), eps, 0.0)
        close(w[0], want[0][0], ep[0], "param"), close(x[2][0], want[1][0], em[0], "m"), close(x[3][0], want[2][0], ev[0], "v")
        assert torch.isfinite(w).all() and np.abs(np.linalg.norm(f64(w), axis=1) - 1).max() <= 16 * U
        return
    v = 0.01 * grad * grad
    tiny = 2.0 ** -148
    step = lambda v: 1e-3 * np.abs(grad) / (np.sqrt(np.maximum(v, 0)) / np.sqrt(0.01) + eps)  # noqa: E731
    low, high = step(v * (1 + 64 * U) + tiny) * (1 - 128 * U), step(v * (1 - 64 * U) - tiny) * (1 + 128 * U)
    moved = np.abs(b - f64(w))
    slack = 2 * U * np.abs(b)
    assert np.all(moved >= low - slack) and np.all(moved <= high + slack)


@gpu
def test_results_do_not_depend_on_alignment():
    """The fast path for aligned tensors and the general one give the same bits, also next to a NaN."""
    for dtype, grad_dtype, master in KINDS:
        a, b = (make((5000,), dtype, 3, master, grad_dtype, off) for off in (0, 1))
        for x in (a, b):
            optim.adamw_step(*[[t] for t in x[:4]], steps_in(5), lr=1e-3, masters=[x[4]])
        assert all(torch.equal(s, t) for s, t in zip(a[:4], b[:4]))
        a, b = (make8((5000,), dtype, 3, master, off) for off in (0, 1))
        for x in (a, b):
            x[1][[700, 701, 4000]] = math.nan
            for _ in range(2):
                optim.adamw8_step(*[[t] for t in x[:6]], steps_in(5), lr=1e-3, masters=[x[6]])
        assert all(torch.equal(s.view(torch.uint8) if s.dtype in optim.STATE8_DTYPES else s.nan_to_num(7.0),
                               t.view(torch.uint8) if t.dtype in optim.STATE8_DTYPES else t.nan_to_num(7.0)) for s, t in zip(a[:6], b[:6]))
        a, b = (make((40, 128), dtype, 3, master, grad_dtype, off) for off in (0, 1))
        for x in (a, b):
            optim.adamw_unit_rows_step(*[[t] for t in x[:4]], steps_in(5), lr=1e-3, masters=[x[4]])
        for s, t in zip(a[:4], b[:4]):                      # the sums over a row are taken in another order
            assert torch.allclose(s.float(), t.float(), rtol=1e-2 if s.dtype != torch.float32 else 1e-4, atol=1e-6)


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_tensors_of_more_than_two_to_the_31_elements(bits):
    """Every kind of offset passes 32 bits; the first, the middle and the last elements are the oracle's."""
    n = 2 ** 31 + 256 * 9 + 77
    g = torch.Generator(device="cuda").manual_seed(1)
    spots = [0, 2 ** 30 - 512, 2 ** 31 - 512, n - 77 - 1024]          # multiples of 256
    p, grad = (torch.zeros(n, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    if bits == 32:
        state = [torch.zeros(n, device="cuda") for _ in range(2)]
    else:
        state = [torch.zeros(n, dtype=d, device="cuda") for d in optim.STATE8_DTYPES]
        scale = [torch.zeros(optim.state8_blocks(n), device="cuda") for _ in range(2)]
    for s in spots:
        p[s:s + 1024] = torch.randn(min(1024, n - s), generator=g, device="cuda").bfloat16()
        grad[s:s + 1024] = torch.randn(min(1024, n - s), generator=g, device="cuda").bfloat16()
    grad[-77:] = torch.randn(77, generator=g, device="cuda").bfloat16()
    parts = [(s, min(s + 1024, n)) for s in spots] + [(n - 77, n)]
    before = [(f64(p[a:b]), grad[a:b].float().cpu().numpy()) for a, b in parts]
    norm = optim.grad_norm([grad])
    want = math.sqrt(sum(float((x[1].astype(np.float64) ** 2).sum()) for x in before))
    assert abs(float(norm) - want) <= NORM_TOL * want
    step = steps_in(0)
    if bits == 32:
        optim.adamw_step([p], [grad], [state[0]], [state[1]], step, lr=1e-2)
    else:
        optim.adamw8_step([p], [grad], [state[0]], [scale[0]], [state[1]], [scale[1]], step, lr=1e-2, seed=11)
    for (a, b), (q, x) in zip(parts, before):
        zero = np.zeros(b - a)
        exact = orc.adamw(q, x, zero, zero, 1, 1e-2)
        bound = bounds((q, x, zero, zero), exact, 1, 1e-2, (0.9, 0.999), 1e-8, 1.0)
        check_params(p[a:b], None, exact[0], bound[0], torch.bfloat16)
        if bits == 32:
            close(state[0][a:b], exact[1], bound[1], "m"), close(state[1][a:b], exact[2], bound[2], "v")
        else:
            blocks = slice(a // 256, -(-b // 256))
            none, nothing = np.zeros(b - a, dtype=np.uint8), np.zeros(-(-(b - a) // 256), dtype=np.float32)
            _, _, m8, ms, v8, vs = orc.adamw8_states(x, none, nothing, none, nothing, 1, 11, 0, first=a)
            assert np.array_equal(bytes_of(state[0][a:b]), m8) and np.array_equal(bytes_of(state[1][a:b]), v8)
            assert np.array_equal(scale[0][blocks].cpu().numpy(), ms) and np.array_equal(scale[1][blocks].cpu().numpy(), vs)


# ---- GPU: unit rows -------------------------------------------------------------------------------------
def rows_bounds(b, want, t, lr, clip, betas=(0.9, 0.999), eps=1e-8, decay=0.01):
    """As ``bounds``, for the row form.  A sum over a row is off by at most (8 + 10 + 1) u of the sum of its absolute terms
    (eight in a row, five and five levels of a tree), so the projection moves g by (40 u) |along|abs |p| + 3 u of its own terms;
    a new row is divided by its length (12 u of the row, and the errors of its elements once more through the length)."""
    p, g, m, v = b
    g = g * clip
    square = np.sum(p * p, axis=1, keepdims=True)
    along = np.divide(np.sum(np.abs(g * p), axis=1, keepdims=True), square, out=np.zeros_like(square), where=square > 0)
    eg = U * (48 * along * np.abs(p) + 8 * np.abs(g))
    projected = np.abs(g) + along * np.abs(p)
    em = U * (3 * betas[0] * np.abs(m) + 4 * (1 - betas[0]) * projected) + (1 - betas[0]) * eg
    ev = U * (3 * betas[1] * np.abs(v) + 5 * (1 - betas[1]) * projected ** 2) + (1 - betas[1]) * (2 * projected * eg + eg * eg)
    # errors of the step, to first order around the exact moments, the denominator at its smallest
    denom = np.sqrt(np.maximum(want[2] - ev, 0)) / math.sqrt(1 - betas[1] ** t) + eps
    rate = lr / (1 - betas[0] ** t)
    upper = np.sqrt(want[2] + ev) / math.sqrt(1 - betas[1] ** t) + eps
    ep = 4 * U * np.abs(p) + rate * (np.abs(want[1]) * (1 / denom - 1 / upper) + em / denom) + 24 * U * rate * np.abs(want[1]) / denom
    new = p * (1 - lr * decay) - rate * want[1] / (np.sqrt(want[2]) / math.sqrt(1 - betas[1] ** t) + eps)
    length = np.sqrt(np.sum(new * new, axis=1, keepdims=True))
    length = np.where(length > 0, length, 1)
    through = np.sum(np.abs(want[0]) * ep, axis=1, keepdims=True) / length
    return (ep / length + np.abs(want[0]) * (through + 12 * U)) * 1.01, em + 2.0 ** -149, ev + 2.0 ** -148


@gpu
@pytest.mark.parametrize("dtype,grad_dtype,master", KINDS)
@pytest.mark.parametrize("F,D,offset", [(1, 1, 0), (5, 7, 0), (300, 8, 0), (33, 255, 0), (33, 256, 0), (33, 257, 1), (40, 512, 1), (500, 768, 0), (9, 2304, 0), (3, 8191, 0), (4, 8192, 0),
                                        (500, 3, 0), (777, 5, 1), (130, 16, 0), (65, 40, 0), (70, 100, 0), (300, 641, 0), (601, 777, 0), (20, 2301, 1),
                                        (310, 4095, 0), (305, 4616, 0), (300, 5632, 0), (301, 5640, 0), (299, 7168, 0), (5, 7176, 0), (4, 8185, 0), (4, 8186, 0)])
def test_unit_rows_against_the_oracle(dtype, grad_dtype, master, F, D, offset):
    x = make((F, D), dtype, F + D, master, grad_dtype, offset, spread=False)
    w = x[4] if master else x[0]
    w.copy_(w.float() / w.float().norm(dim=1, keepdim=True))
    if master:
        x[0].copy_(w)
    if F > 3:
        w[1] = 0                                                # a row of zeros, a row without gradient
        x[0][1] = 0
        x[1][2] = 0
    b = [f64(w), f64(x[1]), f64(x[2]), f64(x[3])]
    step, norm = steps_in(20), torch.tensor(2.0, device="cuda")
    optim.adamw_unit_rows_step(*[[t] for t in x[:4]], step, lr=1e-3, masters=[x[4]] if master else None, norm=norm, max_norm=1.0)
    assert int(step) == 21
    clip = orc.clip_factor(2.0, 1.0)
    want = orc.adamw(*b, 21, 1e-3, clip=clip, unit_rows=True)
    ep, em, ev = rows_bounds(b, want, 21, 1e-3, clip)
    check_params(x[0], x[4], want[0], ep, dtype)
    close(x[2], want[1], em, "m")
    close(x[3], want[2], ev, "v")


@gpu
def test_unit_rows_of_several_decoders_and_zero_rows():
    xs = [make(s, torch.float32, 60 + k, spread=False) for k, s in enumerate([(10, 64), (0, 64), (7, 1000), (3, 0)])]
    for x in xs:
        x[0].copy_(torch.nn.functional.normalize(x[0], dim=1))
    xs[0][0][4], xs[0][1][4], xs[0][2][4], xs[0][3][4] = 0, 0, 0, 0
    step = steps_in(2)
    optim.adamw_unit_rows_step(*[[x[k] for x in xs] for k in range(4)], step, lr=1e-3)
    assert int(step) == 3
    assert float(xs[0][0][4].abs().max()) == 0
    for x in (xs[0], xs[2]):
        length = x[0].double().norm(dim=1)
        assert bool(((length - 1).abs() <= 16 * U)[torch.arange(len(length), device="cuda") != (4 if x is xs[0] else -1)].all())
    with pytest.raises(nv.FlexSaeNativeError, match="8192"):
        y = make((2, 8200), torch.float32, 1)
        optim.adamw_unit_rows_step(*[[t] for t in y[:4]], step, lr=1e-3)


ROW_KERNELS = [5, 8, 40, 256, 257, 640, 777, 2301, 2304, 5640, 7168, 8192]      # row lengths of every way to read a row


def test_oracle_keeps_nothing_finite_beside_a_nan_in_a_row():
    w = np.ones((3, 4)) / 2
    g = np.ones((3, 4))
    w[0, 1], w[1], g[1, 2] = np.nan, 0, np.nan
    p, m, _ = orc.adamw(w, g, 0 * g, 0 * g, 1, 1e-2, unit_rows=True)
    assert np.isnan(p[:2]).all() and np.isfinite(p[2]).all() and np.isnan(m[0]).all() and np.isnan(m[1]).sum() == 1


@gpu
@pytest.mark.parametrize("dtype,grad_dtype,master", KINDS)
@pytest.mark.parametrize("D", ROW_KERNELS)
def test_unit_rows_nonfinite_values_reach_their_row(dtype, grad_dtype, master, D):
    """A NaN or an infinity in a row's parameter or gradient makes the row's length one, so no element of the row stays a number."""
    F = 9
    x = make((F, D), dtype, D, master, grad_dtype, spread=False)
    w = x[4] if master else x[0]
    w.copy_(w.float() / w.float().norm(dim=1, keepdim=True))
    w[0, D // 2], w[2, D - 1], w[6] = math.nan, math.inf, 0
    x[1][4, 0], x[1][6, D // 2], x[1][7, D - 1] = math.inf, math.nan, -math.inf
    if master:
        x[0].copy_(w)
    b = [f64(w), f64(x[1]), f64(x[2]), f64(x[3])]
    with np.errstate(all="ignore"):
        want = orc.adamw(*b, 21, 1e-3, unit_rows=True)
    optim.adamw_unit_rows_step(*[[t] for t in x[:4]], steps_in(20), lr=1e-3, masters=[x[4]] if master else None)
    hit = np.array([0, 2, 4, 6, 7])
    assert np.isnan(want[0][hit]).all()
    for got in (x[0], x[4]) if master else (x[0],):
        assert np.array_equal(np.isnan(f64(got)), np.isnan(want[0]))
    assert np.array_equal(np.isfinite(f64(x[2])), np.isfinite(want[1]))
    clean = [1, 3, 5, 8]
    ep, em, ev = rows_bounds([a[clean] for a in b], [a[clean] for a in want], 21, 1e-3, 1.0)
    check_params(x[0][clean], x[4][clean] if master else None, want[0][clean], ep, dtype)
    close(x[2][clean], want[1][clean], em, "m")
    close(x[3][clean], want[2][clean], ev, "v")


@gpu
@pytest.mark.parametrize("dtype,grad_dtype,master", [k for k in KINDS if k[0] != torch.float16 or k[2]])
@pytest.mark.parametrize("D", ROW_KERNELS)
def test_unit_rows_of_any_length(dtype, grad_dtype, master, D):
    """Rows from 2^-55 to 2^64 long are stepped like others (at 2^-54, 8192 squares lose at most 8192 * 2^-150 = 2^-137 of a sum of
    2^-108).  Shorter ones count as zeros, so that a new row is off by the old one, divided by its length; without a gradient
    they only decay, to two roundings.  Longer ones are left as they were."""
    lengths = [1.0, 2.0 ** 63, 1e12, 1e-8, 2.0 ** -54, 2.0 ** -54, 1e-25, 1e-38, 1e-25, 2.0 ** 66, 1e25, 1e37, 1e37]
    F, still, short, long = len(lengths), [5, 8, 12], [6, 7, 8], [9, 10, 11, 12]
    x = make((F, D), dtype, D + 1, master, grad_dtype, spread=False)
    w = x[4] if master else x[0]
    r = torch.nn.functional.normalize(torch.randn(F, D, dtype=torch.float64, generator=torch.Generator().manual_seed(D)), dim=1)
    w.copy_(r * torch.tensor(lengths, dtype=torch.float64)[:, None])
    if master:
        x[0].copy_(w)
    for k in (1, 2):
        x[k][still] = 0
    before = [t.clone() for t in x if t is not None]
    b = [f64(w), f64(x[1]), f64(x[2]), f64(x[3])]
    old = np.abs(b[0])
    b[0][short] = 0
    want = list(orc.adamw(*b, 21, 1e-3, unit_rows=True))
    optim.adamw_unit_rows_step(*[[t] for t in x[:4]], steps_in(20), lr=1e-3, masters=[x[4]] if master else None)
    for got, was in zip([t for t in x if t is not None], before):
        assert torch.equal(got[long], was[long])
    ep, em, ev = rows_bounds(b, want, 21, 1e-3, 1.0)
    new = -1e-3 / (1 - 0.9 ** 21) * want[1] / (np.sqrt(want[2]) / math.sqrt(1 - 0.999 ** 21) + 1e-8)
    ep[6:8] += old[6:8] / np.sqrt(np.sum(new[6:8] ** 2, axis=1, keepdims=True))
    want[0][8] = f64(before[-1] if master else before[0])[8] * (1 - 1e-3 * 0.01)
    ep[8] = 4 * U * old[8]
    rows = list(range(9))
    check_params(x[0][rows], x[4][rows] if master else None, want[0][rows], ep[rows], dtype)
    close(x[2][rows], want[1][rows], em[rows], "m")
    close(x[3][rows], want[2][rows], ev[rows], "v")


@gpu
@pytest.mark.parametrize("D", ROW_KERNELS)
def test_unit_rows_whose_product_with_the_gradient_overflows(D):
    """Sums over a row are 32-bit: D products of 2e38 / sqrt(D) are sqrt(D) 2e38, past 2^128 from D = 3 on.  The row counts as one with
    an infinity, its neighbours do not notice, and with a clipping factor the same gradient is an ordinary one."""
    w = torch.full((4, D), D ** -0.5, device="cuda")
    g = torch.randn(4, D, generator=torch.Generator().manual_seed(D)).cuda()
    g[1] = 2e38
    zeros = [torch.zeros(4, D, device="cuda") for _ in range(4)]
    first, second = w.clone(), w.clone()
    optim.adamw_unit_rows_step([first], [g], zeros[:1], zeros[1:2], steps_in(0), lr=1e-3)
    assert bool(torch.isnan(first[1]).all()) and bool(torch.isfinite(first[[0, 2, 3]]).all())
    optim.adamw_unit_rows_step([second], [g], zeros[2:3], zeros[3:], steps_in(0), lr=1e-3, norm=torch.tensor(1e30, device="cuda"), max_norm=1.0)
    assert float((second.double().norm(dim=1) - 1).abs().max()) <= 16 * U


# ---- GPU: streams, graphs, versions --------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_replay_like_eager_ones(bits):
    """The step count, the learning rate and the clipping factor are read on the device at every replay."""
    def train(captured):
        g = torch.Generator().manual_seed(3)
        ps = [torch.nn.Parameter(torch.randn(s, generator=g).cuda()) for s in ((70, 33), (33,))]
        lr = torch.tensor(1e-2, device="cuda")
        opt = optim.AdamW(ps, lr=lr, state_bits=bits, max_norm=0.5)
        for p in ps:
            p.grad = torch.randn(p.shape, generator=g).cuda()
        graph = None
        for k in range(6):
            lr.fill_(1e-2 / (k + 1))
            if captured and k == 2:
                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    opt.step()
            if graph is not None:
                graph.replay()
            else:
                opt.step()
            for p in ps:
                p.grad.mul_(-0.7)
        return [p.detach().clone() for p in ps] + [opt.state[ps[0]]["step"].clone()]

    for a, b in zip(train(False), train(True)):
        assert torch.equal(a, b)


@gpu
def test_a_capture_that_would_make_or_split_states_is_refused():
    """States made inside a capture would be set to zero by every replay, a step count split there copied by each."""
    ps = [torch.nn.Parameter(torch.ones(300, device="cuda")) for _ in range(2)]
    opt = optim.AdamW(ps, lr=1e-2)
    for p in ps:
        p.grad = torch.ones_like(p)

    def capture():
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            opt.step()
        return graph

    with pytest.raises(RuntimeError, match="before a step is captured"):
        capture()
    assert not any(opt.state.get(p) for p in ps)
    opt.step()
    ps[1].grad = None
    with pytest.raises(RuntimeError, match="no gradient"):
        capture()
    assert opt.state[ps[0]]["step"] is opt.state[ps[1]]["step"]
    ps[1].grad = torch.ones_like(ps[1])
    graph = capture()
    for _ in range(3):
        graph.replay()
    assert int(opt.state[ps[0]]["step"]) == 4 and torch.equal(ps[0], ps[1])


@gpu
def test_groups_of_one_seed_round_independently_and_masters_come_with_a_foreign_state():
    p, q = (torch.nn.Parameter(torch.zeros(1 << 16, device="cuda")) for _ in range(2))
    opt = optim.AdamW([{"params": [p]}, {"params": [q]}], lr=1e-3, state_bits=8, seed=5)
    for x in (p, q):
        x.grad = torch.randn(1 << 16, generator=torch.Generator().manual_seed(0)).cuda()
    opt.step()
    same = (opt.state[p]["exp_avg"].view(torch.uint8) == opt.state[q]["exp_avg"].view(torch.uint8)).float().mean()
    assert torch.equal(p, q) and 0.3 < float(same) < 0.95             # rounded apart: alike with probability q^2 + (1 - q)^2, 2/3 on average
    a = torch.nn.Parameter(torch.randn(100, device="cuda").bfloat16())
    a.grad = torch.randn_like(a)
    theirs, ours = torch.optim.AdamW([a], lr=1e-3), optim.AdamW([a], lr=1e-3, master_weights=True)
    theirs.step()
    ours.load_state_dict(theirs.state_dict())
    assert torch.equal(ours.state[a]["master"], a.detach().float())
    ours.step()
    assert torch.equal(ours.state[a]["master"].bfloat16(), a.detach())


@gpu
def test_first_call_of_a_process_may_be_captured():
    """Nothing has to be warmed up: every kernel is first launched inside the capture."""
    import subprocess
    import sys

    code = """
import torch
from flexsae_b200 import optim
ts = [[torch.ones(40, 64, device='cuda') for _ in range(2)] for _ in range(4)]
big = torch.ones(1 << 20, device='cuda')
m8 = [torch.zeros(40, 64, dtype=d, device='cuda') for d in optim.STATE8_DTYPES]
s8 = [torch.zeros(10, device='cuda') for _ in range(2)]
step = torch.zeros((), dtype=torch.int64, device='cuda')
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    norm = optim.grad_norm(ts[1] + [big])
    small = optim.grad_norm(ts[1])
    optim.adamw_step(*ts, step, lr=1e-3, norm=norm, max_norm=1.0)
    optim.adamw_unit_rows_step(*ts, step, lr=1e-3, norm=small, max_norm=1.0)
    optim.adamw8_step(ts[0], ts[1], [m8[0], m8[0].clone()], [s8[0], s8[0].clone()], [m8[1], m8[1].clone()], [s8[1], s8[1].clone()], step, lr=1e-3)
for _ in range(3):
    graph.replay()
torch.cuda.synchronize()
assert int(step) == 9 and abs(float(norm) - (2 * 2560 + (1 << 20)) ** 0.5) < 1e-3 and abs(float(small) - 5120 ** 0.5) < 1e-4
print('captured')
"""
    import os

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stdout + r.stderr


@gpu
def test_two_captured_graphs_replay_side_by_side():
    """Two graphs captured one after the other from the same stream hold their own scratch memory."""
    sets = [make((3000, 333), torch.bfloat16, 70 + k) for k in range(2)]
    grads = [[x[1], torch.randn(1 << 20, generator=torch.Generator().manual_seed(k)).cuda()] for k, x in enumerate(sets)]
    steps, want = [steps_in(0), steps_in(0)], []
    for k, x in enumerate(sets):
        y = [t.clone() for t in x[:4]]
        count = steps_in(0)
        for _ in range(8):
            norm = optim.grad_norm(grads[k])
            optim.adamw_step(*[[t] for t in y], count, lr=1e-3, norm=norm, max_norm=1.0)
        want.append(y)
    graphs = []
    for k, x in enumerate(sets):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            norm = optim.grad_norm(grads[k])
            optim.adamw_step(*[[t] for t in x[:4]], steps[k], lr=1e-3, norm=norm, max_norm=1.0)
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(8):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for x, y, count in zip(sets, want, steps):
        assert int(count) == 8 and all(torch.equal(a, b) for a, b in zip(x[:4], y))


@gpu
def test_steps_on_two_streams_do_not_disturb_each_other():
    def run(streams):
        sets = [make((4000, 257), torch.float32, 20 + k) for k in range(2)]
        steps, norms = [steps_in(0), steps_in(0)], [None, None]
        torch.cuda.synchronize()
        for _ in range(5):
            for k in range(2):
                with torch.cuda.stream(streams[k]):
                    norms[k] = optim.grad_norm([sets[k][1]])
                    optim.adamw_step(*[[t] for t in sets[k][:4]], steps[k], lr=1e-3, norm=norms[k], max_norm=1.0)
        torch.cuda.synchronize()
        return [t for x in sets for t in (x[0], x[2], x[3])] + steps

    one = torch.cuda.current_stream()
    for a, b in zip(run([one, one]), run([torch.cuda.Stream(), torch.cuda.Stream()])):
        assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("entry", ["norm", "adamw", "adamw8", "rows"])
def test_calls_wait_for_the_copies_and_fills_before_them(entry):
    """Launches are set up early; what they read may still be on its way, from the host, on the device or from another stream."""
    F, D = 6000, 4096
    host = torch.randn(F, D, generator=torch.Generator().manual_seed(3)).pin_memory()
    source = host.cuda()
    side = torch.cuda.Stream()

    def run(bring):
        p, grad = torch.ones(F, D, device="cuda"), torch.full((F, D), 7.0, device="cuda")
        m, v = (torch.zeros(F, D, device="cuda") for _ in range(2))
        m8, v8 = (torch.zeros(F, D, dtype=d, device="cuda") for d in optim.STATE8_DTYPES)
        scales = [torch.zeros(F * D // 256, device="cuda") for _ in range(2)]
        step = steps_in(0)
        torch.cuda.synchronize()
        bring(grad)
        if entry == "norm":
            out = [optim.grad_norm([grad])]
        elif entry == "adamw8":
            optim.adamw8_step([p], [grad], [m8], [scales[0]], [v8], [scales[1]], step, lr=1e-2)
            out = [p, m8.view(torch.uint8), scales[1]]
        else:
            (optim.adamw_step if entry == "adamw" else optim.adamw_unit_rows_step)([p], [grad], [m], [v], step, lr=1e-2)
            out = [p, m, v]
        grad.fill_(math.nan)                     # and what follows waits for them
        torch.cuda.synchronize()
        return out

    def from_side(grad):
        with torch.cuda.stream(side):
            grad.copy_(source)
        torch.cuda.current_stream().wait_stream(side)

    def zeroed(grad):
        grad.zero_()
        grad.add_(source)

    want = run(lambda grad: (grad.copy_(source), torch.cuda.synchronize()))
    for bring in (lambda grad: grad.copy_(host, non_blocking=True), lambda grad: grad.copy_(source), from_side, zeroed):
        assert all(torch.equal(a, b) for a, b in zip(run(bring), want))
    cleared = run(lambda grad: grad.zero_())
    if entry == "norm":
        assert float(cleared[0]) == 0


@gpu
def test_autograd_sees_that_a_parameter_changed():
    p = torch.randn(8, device="cuda", requires_grad=True)
    loss = (p * p).sum()
    optim.adamw_step([p], [torch.ones(8, device="cuda")], [torch.zeros(8, device="cuda")], [torch.zeros(8, device="cuda")], steps_in(0), lr=1e-3)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@gpu
def test_every_tensor_that_a_step_writes_counts_a_version():
    p, g, _, _, w = make((16, 32), torch.bfloat16, 3, master=True)
    m, v = (torch.zeros(16, 32, device="cuda").to(d) for d in optim.STATE8_DTYPES)
    scales, step, norm = [torch.zeros(2, device="cuda") for _ in range(2)], steps_in(0), optim.grad_norm([g])
    tensors = [p, w, m, v, *scales, step, g, norm]
    before = [t._version for t in tensors]
    optim.adamw8_step([p], [g], [m], [scales[0]], [v], [scales[1]], step, lr=1e-3, masters=[w], norm=norm)
    assert [t._version - k for t, k in zip(tensors, before)] == [1] * 7 + [0] * 2


# ---- GPU: the optimizer class, and a training run -----------------------------------------------------------
def make_sae(F, D, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    w = torch.nn.functional.normalize(torch.randn(F, D, generator=g), dim=1)
    return {k: torch.nn.Parameter(t.to(dtype).cuda()) for k, t in
            dict(w_enc=w.clone(), b_enc=torch.zeros(F), w_dec=w, b_dec=torch.zeros(D)).items()}


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits,master", [(32, False), (32, True), (8, False), (8, True)])
def test_training_run_encoder_selection_loss_and_step(dtype, bits, master):
    """Encoder, top-K selection, fused loss, its backward and the optimizer step together, four times: every step is what
    the oracle makes of the gradients that the losses left, clipped by their norm, and the decoder's rows stay at
    unit length."""
    import flexsae_b200 as fx
    from flexsae_b200 import producer

    F, D, K, B, lr, max_norm = 512, 128, 16, 96, 1e-3, 0.05
    sae = make_sae(F, D, dtype)
    opt = optim.AdamW([{"params": [sae["w_enc"], sae["b_enc"], sae["b_dec"]], "state_bits": bits, "seed": 9},
                       {"params": [sae["w_dec"]], "unit_rows": True}], lr=lr, eps=1e-6, max_norm=max_norm, master_weights=master)
    held = master and dtype != torch.float32
    m = {k: np.zeros(tuple(p.shape)) for k, p in sae.items()}
    v = {k: np.zeros(tuple(p.shape)) for k, p in sae.items()}
    for t in range(1, 5):
        x = torch.randn(B, D, generator=torch.Generator().manual_seed(50 + t)).to(dtype).cuda()
        idx, vals = producer.encode_topk(x - sae["b_dec"], sae["w_enc"], sae["b_enc"], K)
        fx.triton_hierarchical_sae_loss(idx, sae["w_dec"], vals, sae["b_dec"], x).backward()
        grads = {k: f64(p.grad) for k, p in sae.items()}
        before = {k: f64(opt.state[p]["master"] if held and t > 1 else p) for k, p in sae.items()}
        opt.step()
        norm = math.sqrt(sum(float((g * g).sum()) for g in grads.values()))
        assert abs(float(opt.norm) - norm) <= NORM_TOL * norm
        clip = orc.clip_factor(float(opt.norm), max_norm)
        for k, p in sae.items():
            rows = k == "w_dec"
            want = orc.adamw(before[k], grads[k], m[k], v[k], t, lr, eps=1e-6, clip=clip, unit_rows=rows)
            state = opt.state[p]
            assert int(state["step"]) == t
            if rows or bits == 32:
                b = (before[k], grads[k], m[k], v[k])
                ep, em, ev = rows_bounds(b, want, t, lr, clip, eps=1e-6) if rows else bounds(b, want, t, lr, (0.9, 0.999), 1e-6, clip)
                close(state["exp_avg"], want[1], em, k)
                close(state["exp_avg_sq"], want[2], ev, k)
                m[k], v[k] = f64(state["exp_avg"]), f64(state["exp_avg_sq"])
            else:
                # the parameter from moments off by the bounds above; here the 8-bit states are only read back
                ep = bounds((before[k], grads[k], m[k], v[k]), want, t, lr, (0.9, 0.999), 1e-6, clip)[0]
                m[k], v[k] = (f64(state[n].float().reshape(-1) * state[n + "_scale"].repeat_interleave(256)[: p.numel()]).reshape(tuple(p.shape))
                              for n in ("exp_avg", "exp_avg_sq"))
            check_params(p, state.get("master"), want[0], ep, dtype)
        opt.zero_grad()
    length = sae["w_dec"].double().norm(dim=1)
    assert float((length - 1).abs().max()) <= (16 * U if dtype == torch.float32 else 2.0 ** -8)


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict_continues_the_run(bits):
    def params():
        return [torch.nn.Parameter(p.detach().clone()) for p in make_sae(64, 40, torch.bfloat16).values()]

    def grads(ps, t):
        g = torch.Generator().manual_seed(t)
        for p in ps:
            p.grad = torch.randn(p.shape, generator=g).to(p.dtype).cuda()

    kw = dict(lr=1e-2, state_bits=bits, master_weights=True, seed=4)
    a, b = params(), params()
    first, second = optim.AdamW(a, **kw), optim.AdamW(b, **kw)
    for t in range(3):
        grads(a, t)
        first.step()
    with torch.no_grad():
        for p, q in zip(a, b):
            q.copy_(p)
    second.load_state_dict(first.state_dict())
    for p, q in zip(a, b):
        for name, value in first.state[p].items():
            assert second.state[q][name].dtype == value.dtype and second.state[q][name].data_ptr() != value.data_ptr()
    for t in range(3, 5):
        grads(a, t), grads(b, t)
        first.step(), second.step()
    assert len({id(second.state[q]["step"]) for q in b}) == 1
    for p, q in zip(a, b):
        assert torch.equal(p, q)
        for name, value in first.state[p].items():
            assert torch.equal(value.view(torch.uint8) if value.dim() else value, second.state[q][name].view(torch.uint8) if value.dim() else second.state[q][name])


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_state_of_torchs_adamw_is_taken_over(dtype):
    ps, qs = ([torch.nn.Parameter(p.detach().clone()) for p in make_sae(64, 40, dtype).values()] for _ in range(2))
    theirs, ours = torch.optim.AdamW(ps, lr=1e-2), optim.AdamW(qs, lr=5e-3, max_norm=1e9)
    for t in range(3):
        for p in ps:
            p.grad = torch.randn(p.shape, generator=torch.Generator().manual_seed(t)).to(dtype).cuda()
        theirs.step()
    with torch.no_grad():
        for p, q in zip(ps, qs):
            q.copy_(p)
            q.grad = p.grad.clone()
    ours.load_state_dict(theirs.state_dict())
    assert ours.param_groups[0]["lr"] == 1e-2 and ours.param_groups[0]["state_bits"] == 32
    before = [[f64(t) for t in (q, q.grad, ours.state[q]["exp_avg"], ours.state[q]["exp_avg_sq"])] for q in qs]
    ours.step()
    for q, b in zip(qs, before):
        want = orc.adamw(*b, 4, 1e-2)
        ep, em, ev = bounds(b, want, 4, 1e-2, (0.9, 0.999), 1e-8, 1.0)
        assert int(ours.state[q]["step"]) == 4 and ours.state[q]["exp_avg"].dtype == torch.float32
        check_params(q, None, want[0], ep, dtype)
        close(ours.state[q]["exp_avg"], want[1], em, "m"), close(ours.state[q]["exp_avg_sq"], want[2], ev, "v")


@gpu
def test_parameters_without_gradients_keep_their_own_count():
    ps = [torch.nn.Parameter(torch.ones(300, device="cuda")) for _ in range(3)]
    opt = optim.AdamW(ps, lr=1e-2)
    counts = [0, 0, 0]
    for t, active in enumerate([(0, 1), (0, 1, 2), (1,), (0, 2), (0, 1, 2)]):
        for k, p in enumerate(ps):
            p.grad = torch.full_like(p, 0.1 * (t + 1)) if k in active else None
        kept = [p.detach().clone() for p in ps]
        opt.step()
        for k, p in enumerate(ps):
            counts[k] += k in active
            assert torch.equal(p, kept[k]) == (k not in active)
            assert (int(opt.state[p]["step"]) if opt.state.get(p) else 0) == counts[k]


@gpu
def test_skip_nonfinite_and_copies_of_the_optimizer():
    import copy
    import pickle

    p = torch.nn.Parameter(torch.ones(300, device="cuda"))
    opt = optim.AdamW([p], lr=1e-2, skip_nonfinite=True)
    p.grad = torch.ones_like(p)
    opt.step()
    kept = p.detach().clone()
    p.grad[7] = math.inf
    opt.step()
    assert torch.equal(p, kept) and int(opt.state[p]["step"]) == 1 and float(opt.norm) == math.inf
    for other in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        q = other.param_groups[0]["params"][0]
        q.grad = torch.ones_like(q)
        other.step()
        assert other.skip_nonfinite and int(other.state[q]["step"]) == 2 and not torch.equal(q, kept)


@gpu
@pytest.mark.parametrize("optimizer", ["adamw", "adamw8", "unit_rows"])
def test_example_times_a_training_step(optimizer, capsys):
    from flexsae_b200 import example

    r = example.main(["--B", "64", "--K", "32", "--F", "1024", "--D", "256", "--iters", "2", "--warmup", "1", "--optimizer", optimizer])
    assert 0 < r["training"]["fused_optimizer"] < r["training"]["fused"] and r["training"]["torch"] > 0
    assert "training step" in capsys.readouterr().out
