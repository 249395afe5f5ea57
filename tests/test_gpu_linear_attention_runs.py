"""Linear attention, the prompt conv and the gated norm as they are run: many and
long sequences, padded batches, graphs that replay, streams, memory shared by
calls (bounds in tests/linear_util.py)."""
import pytest
import torch

from muserve_amd.kernels import linear_attention as la
from muserve_amd.state_pool import StatePool
from oracle import linear as ref
from tests import linear_util as lu
from tests.gpu_util import DEV, case
from tests.test_gpu_linear_attention import check_prompts, ints, prompt, step

pytestmark = pytest.mark.gpu
D = 128


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("hk,hv", [(1, 9), (3, 3), (2, 22), (5, 10)])
def test_head_groups(hk, hv, delta):
    case(f"linear attention prompts, {hk}/{hv} heads, delta {delta}")
    x = lu.inputs(hv, 75, hk, hv, slots=3, delta=delta, wide=True)
    check_prompts(x, [66, 9], [2, 0])


@pytest.mark.parametrize("delta", [True, False])
def test_a_long_prompt(delta):
    """Long enough to be cut into segments, behind short ones."""
    case(f"linear attention prompts of 20, 2600 and 700 tokens, delta {delta}")
    x = lu.inputs(11, 3325, 1, 2, slots=3, delta=delta, norm=True)
    check_prompts(x, [20, 2600, 700], [1, 0, 2], norm=True, first=2, max_seqlen=2600)


@pytest.mark.parametrize("longest", [None, 9])
def test_many_sequences(longest):
    """600 sequences of 0 to 9 tokens (some of them empty and without a slot)."""
    case(f"linear attention over 600 short prompts, max_seqlen {longest}")
    gen = torch.Generator().manual_seed(4)
    lens = torch.randint(0, 10, (600,), generator=gen).tolist()
    x = lu.inputs(13, sum(lens) + 3, 1, 2, slots=640)
    slots = torch.randperm(640, generator=gen)[:600].tolist()
    check_prompts(x, lens, slots, first=1, max_seqlen=longest)


def test_many_sequences_token_by_token():
    case("linear attention over 600 prompts of up to 8 tokens")
    gen = torch.Generator().manual_seed(5)
    lens = torch.randint(0, 9, (600,), generator=gen).tolist()
    x = lu.inputs(14, sum(lens), 1, 2, slots=600, norm=True)
    check_prompts(x, lens, list(range(600)), norm=True, max_seqlen=8)


@pytest.mark.parametrize("longest", [8, 70, 1300])
def test_padded_batches(longest):
    """Empty sequences at the end of a batch need no slot and raise nothing."""
    case(f"linear attention and conv, padded batch, up to {longest} tokens")
    lens = [longest, 3]
    total = sum(lens)
    x = lu.inputs(6, total + 5, 2, 8, slots=2)
    gx = lu.on_gpu(x)
    cu, slots = ints([0, longest, total, total, total]), ints([1, 0, -1, -1])
    states = [gx["state"].clone(), gx["state"].clone()]
    outs = [torch.full((total + 5, 8, D), 7.0, device=DEV).bfloat16() for _ in range(2)]
    prompt(gx, slots, cu, states[0], out=outs[0], max_seqlen=longest)
    prompt(gx, slots[:2], cu[:3], states[1], out=outs[1], max_seqlen=longest)
    w = torch.randn(64, 4, device=DEV).bfloat16()
    rows, conv = torch.randn(total + 5, 64, device=DEV).bfloat16(), torch.randn(2, 64, 4, device=DEV)
    convs = [conv.bfloat16(), conv.bfloat16()]
    ys = [torch.full((total + 5, 64), 7.0, device=DEV).bfloat16() for _ in range(2)]
    la.causal_conv_prefill(rows, w, convs[0], slots, cu, out=ys[0])
    la.causal_conv_prefill(rows, w, convs[1], slots[:2], cu[:3], out=ys[1])
    la.check_errors(DEV)
    assert torch.equal(outs[0], outs[1]) and torch.equal(states[0], states[1])
    assert torch.equal(ys[0], ys[1]) and torch.equal(convs[0], convs[1])
    assert (outs[0][total:] == 7).all() and (ys[0][total:] == 7).all()


@pytest.mark.parametrize("lens", [[3, 8], [200, 65], [5000, 300]], ids=str)
def test_same_bits_every_time(lens):
    case(f"linear attention prompts {lens}, twice")
    x = lu.on_gpu(lu.inputs(7, sum(lens), 2, 8, norm=True, slots=2))
    runs = []
    for _ in range(2):
        state = x["state"].clone()
        out = prompt(x, ints([0, 1]), ints([0, lens[0], sum(lens)]), state, max_seqlen=max(lens))
        runs.append((out, state))
    la.check_errors(DEV)
    assert torch.equal(runs[0][0], runs[1][0]) and torch.equal(runs[0][1], runs[1][1])


@pytest.mark.parametrize("delta", [True, False])
def test_nan_in_a_segment(delta):
    """A NaN value of a long prompt that is cut into segments reaches its value
    dim of its head, from its token on, and nothing else."""
    case(f"linear attention, NaN inside a long prompt, delta {delta}")
    T, at, hk, hv = 6000, 3333, 1, 4
    x = lu.inputs(15, T, hk, hv, delta=delta)
    clean = lu.on_gpu(x)
    x["mixed"][at, 2 * hk * D + 2 * D + 17] = float("nan")
    dirty = lu.on_gpu(x)
    runs = []
    for y in (clean, dirty):
        state = y["state"].clone()
        runs.append((prompt(y, ints([0]), ints([0, T]), state).float(), state))
    la.check_errors(DEV)
    (want, w_state), (got, g_state) = runs
    # A chunk of 64 tokens with a NaN is walked token by token by the wave that has
    # it (16 value dims), its tokens before the NaN too: there the fp32 results of
    # two ways of summing are each rounded to bf16, by 2^-8 of a value each, so the
    # two differ by 2^-7 of its size (in the norm over values; the sums' own 2^-20
    # or so vanish beside it).
    start = at // 64 * 64
    assert torch.equal(got[:start], want[:start])
    a, b = got[start:at, 2, 16:32].double(), want[start:at, 2, 16:32].double()
    assert (a - b).norm() <= 2.0 ** -7 * b.norm()
    same = [i for i in range(D) if not 16 <= i < 32]
    assert torch.equal(got[start:, 2][:, same], want[start:, 2][:, same])
    for h in (0, 1, 3):
        assert torch.equal(got[:, h], want[:, h]) and torch.equal(g_state[0, h], w_state[0, h])
    assert not torch.isfinite(got[at:, 2, 17]).any()
    others = [i for i in range(D) if i != 17]
    a, b = got[at:, 2][:, others].double(), want[at:, 2][:, others].double()
    assert torch.isfinite(a).all() and (a - b).norm() <= 2.0 ** -7 * b.norm()
    a, b = g_state[0, 2][others].double(), w_state[0, 2][others].double()
    assert torch.isfinite(a).all() and (a - b).norm() <= 1e-5 * b.norm()


def layer(pool, x, proj, w, slots, cu, news):
    """A layer's prompts and then one step for each request; returns all outputs."""
    hk, hv, total = x["hk"], x["hv"], int(x["tokens"])
    how = {n: lu.keywords(x)[n] for n in ("a_log", "dt_bias", "qk_norm")}
    mixed = pool.conv_prefill(0, slots, proj[:total], w, cu)
    o = pool.linear_attn_prefill(0, slots, *lu.split(mixed, hk, hv), x["g"][:total],
                                 x["beta"][:total], cu, z=x["z"][:total], norm_weight=x["w"], **how)
    r = slice(total, total + news)
    step_in = pool.conv_decode(0, slots, proj[r], w)
    p = pool.linear_attn_decode(0, slots, *lu.split(step_in, hk, hv), x["g"][r], x["beta"][r], **how)
    y = la.gated_rms_norm(p, x["z"][r], x["w"])
    return mixed, o, step_in, p, y


@pytest.mark.parametrize("lens", [[4, 2], [90, 33], [4000, 70]], ids=str)
def test_graph_replays(lens):
    """The layer captured once and replayed, with eager work on the same and
    other tensors between the replays, gives what eager calls give."""
    case(f"GDN layer captured and replayed, prompts {lens}")
    hk, hv, news, total = 2, 8, len(lens), sum(lens)
    C = (2 * hk + hv) * D
    x = lu.on_gpu(lu.inputs(21, total + news, hk, hv, norm=True))
    x["tokens"] = total
    gen = torch.Generator().manual_seed(22)
    proj = torch.randn(total + news, C, generator=gen).bfloat16().to(DEV)
    w = (0.5 * torch.randn(C, 4, generator=gen)).bfloat16().to(DEV)
    slots, cu = ints([1, 2]), ints([0, lens[0], total])
    pools = [StatePool(num_layers=1, num_slots=3, conv_shape=(C, 4), device=DEV) for _ in range(2)]
    for p in pools:
        p.reset([0, 1, 2])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(pools[0], x, proj, w, slots, cu, news)
    torch.cuda.current_stream().wait_stream(side)
    for p in pools:
        p.reset([0, 1, 2])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = layer(pools[0], x, proj, w, slots, cu, news)
    for turn in range(4):  # states go on from turn to turn
        proj.mul_(0.9)
        x["g"].add_(0.1)
        graph.replay()
        eager = layer(pools[1], x, proj, w, slots, cu, news)
        other = prompt(x, ints([0]), ints([0, total]), torch.zeros(1, hv, D, D, device=DEV))
        torch.cuda.synchronize()
        for got, want in zip(captured, eager):
            assert torch.equal(got, want), turn
        assert torch.equal(pools[0].state, pools[1].state)
        assert torch.equal(pools[0].conv, pools[1].conv)
        assert torch.isfinite(other[:total].float()).all()  # (rows behind are not written)
    for p in pools:
        p.check_errors()
    la.check_errors(DEV)


def test_two_streams_at_once():
    """Calls in flight on two streams do not meet."""
    case("linear attention on two streams at once")
    xs = [lu.on_gpu(lu.inputs(30 + i, 3000, 2, 8, norm=True)) for i in range(2)]
    cu, slot = ints([0, 3000]), ints([0])
    want = []
    for x in xs:
        state = x["state"].clone()
        want.append((prompt(x, slot, cu, state), state))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(3):
        for x, s in zip(xs, streams):
            with torch.cuda.stream(s):
                state = x["state"].clone()
                got.append((prompt(x, slot, cu, state), state))
    torch.cuda.synchronize()
    la.check_errors(DEV)
    for i, (out, state) in enumerate(got):
        assert torch.equal(out, want[i % 2][0]) and torch.equal(state, want[i % 2][1]), i


def test_ids_of_64_bits_and_lists_with_gaps():
    case("linear attention, slots and offsets in int64 and strided")
    x = lu.on_gpu(lu.inputs(16, 20, 2, 8, slots=4))
    slots, cu = [3, 1], [0, 13, 20]
    states = [x["state"].clone() for _ in range(2)]
    want = prompt(x, ints(slots), ints(cu), states[0])
    wide = torch.tensor([[a, -9] for a in slots], device=DEV)[:, 0]
    got = prompt(x, wide, torch.tensor(cu, device=DEV), states[1])
    assert torch.equal(got, want) and torch.equal(states[0], states[1])
    rows = {n: t[:2] if n in ("mixed", "g", "beta") else t for n, t in x.items()}
    got, want = step(rows, wide, states[0]), step(rows, ints(slots), states[1])
    la.check_errors(DEV)
    assert torch.equal(got, want) and torch.equal(states[0], states[1])


def test_rows_far_apart():
    """Strides of megabytes between the token rows of one buffer."""
    case("linear attention on rows 2 MiB apart")
    T, hk, hv = 70, 1, 2
    x = lu.inputs(17, T, hk, hv)
    buf = torch.zeros(T, 1 << 20, dtype=torch.bfloat16, device=DEV)
    wide = buf[:, 4096:4096 + (2 * hk + hv) * D]
    wide.copy_(x["mixed"])
    x["mixed"] = x["mixed"][:, :(2 * hk + hv) * D]
    gx = lu.on_gpu(x)
    states = [gx["state"].clone() for _ in range(2)]
    want = prompt(gx, ints([0]), ints([0, T]), states[0])
    got = la.linear_attn_prefill(wide[:, :D].view(T, 1, D), wide[:, D:2 * D].view(T, 1, D),
                                 wide[:, 2 * D:].unflatten(1, (hv, D)), gx["g"], gx["beta"], states[1],
                                 ints([0]), ints([0, T]), **lu.keywords(gx))
    la.check_errors(DEV)
    assert torch.equal(got, want) and torch.equal(states[0], states[1])


def test_memory_shared_by_out_and_inputs():
    case("linear attention, conv and norm: out on an input's memory")
    x = lu.on_gpu(lu.inputs(18, 6, 8, 8, norm=True, slots=6))
    q, k, v = (t.contiguous() for t in lu.split(x["mixed"], 8, 8))
    at, cu = ints([0]), ints([0, 6])
    kept = [t.clone() for t in (q, k, v, x["z"], x["state"])]
    arena = torch.zeros(20, 8, D, dtype=torch.bfloat16, device=DEV)
    inside = arena[2:8]
    inside.copy_(v)
    for out, vv in ((q, v), (k, v), (v, v), (x["z"], v), (arena[:6], inside), (arena[7:13], inside)):
        with pytest.raises(ValueError, match="out must not be"):
            la.linear_attn_prefill(q, k, vv, x["g"], x["beta"], x["state"], at, cu, z=x["z"],
                                   norm_weight=x["w"], out=out)
        with pytest.raises(ValueError, match="out must not be"):
            la.linear_attn_decode(q, k, vv, x["g"], x["beta"], x["state"], ints(range(6)), z=x["z"],
                                  norm_weight=x["w"], out=out)
    la.linear_attn_prefill(q, k, inside, x["g"], x["beta"], x["state"].clone(), at, cu,
                           out=arena[8:14])  # next to it
    for t, u in zip((q, k, v, x["z"], x["state"]), kept):
        assert torch.equal(t, u)
    rows = torch.randn(9, 64, device=DEV).bfloat16()
    with pytest.raises(ValueError, match="out must not be x"):
        la.causal_conv_prefill(rows[1:], torch.zeros(64, 4, device=DEV).bfloat16(),
                               torch.zeros(1, 64, 4, device=DEV).bfloat16(), at, ints([0, 8]),
                               out=rows[:8])
    want = la.gated_rms_norm(v, x["z"], x["w"])
    for name in ("x", "z"):
        a, b = v.clone(), x["z"].clone()
        assert torch.equal(la.gated_rms_norm(a, b, x["w"], out=a if name == "x" else b), want)
    with pytest.raises(ValueError, match="out must not be x"):
        la.gated_rms_norm(arena[:6], x["z"], x["w"], out=arena[1:7])
    wide = torch.zeros(6, 8 * D + 64, dtype=torch.bfloat16, device=DEV)
    strided = wide[:, :8 * D].unflatten(1, (8, D))
    with pytest.raises(ValueError, match="out must not be x"):
        la.gated_rms_norm(strided, x["z"], x["w"], out=wide.flatten()[:6 * 8 * D].view(6, 8, D))
    la.check_errors(DEV)


def test_conv_of_many_sequences():
    case("prompt conv of 300 short sequences")
    gen = torch.Generator().manual_seed(40)
    lens = torch.randint(0, 7, (300,), generator=gen).tolist()
    C, total = 72, sum(lens)
    conv = torch.randn(300, C, 4, generator=gen).bfloat16()
    x, w = torch.randn(total, C, generator=gen).bfloat16(), torch.randn(C, 4, generator=gen).bfloat16()
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    gconv = conv.to(DEV)
    out = la.causal_conv_prefill(x.to(DEV), w.to(DEV), gconv, ints(range(300)), ints(cu))
    la.check_errors(DEV)
    for b in range(300):
        rows = slice(cu[b], cu[b + 1])
        want, mass = ref.conv_prompt(conv, b, x[rows], w)
        lu.close(out[rows], want, 2.0 ** -20 * mass, f"sequence {b}")
    assert torch.equal(gconv.cpu(), conv)


@pytest.mark.parametrize("rows,dim", [(70001, 128), (140000, 64), (20000, 504), (4300000, 512)])
def test_norm_of_many_rows(rows, dim):
    case(f"gated norm of {rows} rows of {dim}")
    gen = torch.Generator(device=DEV).manual_seed(rows)
    x, z = (torch.randn(rows, dim, generator=gen, device=DEV).bfloat16() for _ in range(2))
    w = torch.randn(dim, generator=gen, device=DEV)
    got = la.gated_rms_norm(x, z, w)
    some = torch.cat([torch.arange(0, rows, 97), torch.arange(rows - 70, rows)])
    want = ref.gated_norm(x[some].cpu(), z[some].cpu(), w.cpu(), 1e-6)
    lu.close(got[some], want, (64 + dim ** 0.5) * lu.U32 * want.abs(), "rows")


def test_slots_past_32_bits():
    """State and conv pools of more than 4 GiB, used at their far ends."""
    case("linear attention and conv on slots behind 4 GiB")
    hk, hv, pool, C = 1, 2, 36000, 16
    x = lu.inputs(50, 75, hk, hv, slots=2)
    state = torch.empty(pool, hv, D, D, device=DEV)
    assert state.numel() * 4 > 1 << 32
    slots = [pool - 1, 33000]
    gx = lu.on_gpu(x)
    near = gx["state"].clone()
    for longest, cu in ((70, [0, 70, 75]), (5, [0, 3, 8])):
        state[slots] = near
        got = prompt(gx, ints(slots), ints(cu), state, max_seqlen=longest)
        want_state = near.clone()
        want = prompt(gx, ints([0, 1]), ints(cu), want_state, max_seqlen=longest)
        assert torch.equal(got[:cu[-1]], want[:cu[-1]]) and torch.equal(state[slots], want_state)
    rows = {n: t[:2] if n in ("mixed", "g", "beta") else t for n, t in gx.items()}
    got, want = step(rows, ints(slots), state), step(rows, ints([0, 1]), want_state)
    assert torch.equal(got, want) and torch.equal(state[slots], want_state)
    del state
    conv = torch.empty((1 << 25) + 64, C, 4, dtype=torch.bfloat16, device=DEV)
    assert conv.numel() * 2 > 1 << 32
    far = [conv.shape[0] - 1, conv.shape[0] - 9]
    near = torch.randn(2, C, 4, device=DEV).bfloat16()
    conv[far] = near
    y, w = torch.randn(70, C, device=DEV).bfloat16(), torch.randn(C, 4, device=DEV).bfloat16()
    got = la.causal_conv_prefill(y, w, conv, ints(far), ints([0, 68, 70]))
    want = la.causal_conv_prefill(y, w, near, ints([0, 1]), ints([0, 68, 70]))
    la.check_errors(DEV)
    assert torch.equal(got, want) and torch.equal(conv[far], near)


def test_rows_past_32_bits():
    """Rows of v, z and out behind 4 GiB: a short prompt behind a long one gives
    what it gives alone (its walk may be cut otherwise: two roundings to bf16 of
    2^-8 each way, states by what fp32 sums do)."""
    case("linear attention on 300000 tokens of 64 heads")
    T, hk, hv, last = 300000, 1, 64, 90
    gen = torch.Generator(device=DEV).manual_seed(51)

    def normal(*size):
        return torch.randn(*size, generator=gen, device=DEV, dtype=torch.bfloat16)

    q, k, v = normal(T, hk, D), normal(T, hk, D), normal(T, hv, D)
    assert v.numel() * 2 > 1 << 32
    g, beta = -0.1 * normal(T, hv).abs(), torch.sigmoid(normal(T, hv))
    state = torch.zeros(2, hv, D, D, device=DEV)
    w = 1 + 0.1 * normal(D)
    out = la.linear_attn_prefill(q, k, v, g, beta, state, ints([0, 1]), ints([0, T - last, T]),
                                 max_seqlen=T - last, qk_norm=True, z=v, norm_weight=w)
    alone = torch.zeros(1, hv, D, D, device=DEV)
    tail = [t[T - last:] for t in (q, k, v, g, beta)]
    want = la.linear_attn_prefill(*tail, alone, ints([0]), ints([0, last]), max_seqlen=last,
                                  qk_norm=True, z=tail[2], norm_weight=w)
    la.check_errors(DEV)
    assert torch.isfinite(out.float()).all()
    for a, b, tol in ((out[T - last:], want, 2.0 ** -6), (state[1], alone[0], 1e-5)):
        assert (a.double() - b.double()).norm() <= tol * b.double().norm()
    normed = la.gated_rms_norm(v, v, w)
    some = slice(T - 5, T)
    assert torch.equal(normed[some], la.gated_rms_norm(v[some], v[some], w))
    mixed = v.view(T, hv * D)
    cw, conv = normal(hv * D, 4), torch.zeros(2, hv * D, 4, dtype=torch.bfloat16, device=DEV)
    y = la.causal_conv_prefill(mixed, cw, conv, ints([0, 1]), ints([0, T - last, T]))
    conv1 = torch.zeros(1, hv * D, 4, dtype=torch.bfloat16, device=DEV)
    y1 = la.causal_conv_prefill(mixed[T - last:], cw, conv1, ints([0]), ints([0, last]))
    la.check_errors(DEV)
    assert torch.equal(y[T - last:], y1) and torch.equal(conv[1], conv1[0])


@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("delta", [True, False])
def test_heads_of_one_key_head_in_turn(delta, norm):
    """More images than a launch holds, all of one key head: its value heads in turn,
    with a few of them alone as the reference (bounds as for key heads in turn)."""
    case(f"linear attention, 2/192 heads x 70000 tokens in several launches, delta {delta}")
    T, hk, hv = 70000, 2, 192
    gen = torch.Generator(device=DEV).manual_seed(61)

    def normal(*size):
        return torch.randn(*size, generator=gen, device=DEV).bfloat16()

    q, k, v = normal(T, hk, D), normal(T, hk, D), normal(T, hv, D)
    x = {"g": normal(T, hv), "beta": normal(T, hv) if delta else None,
         "z": normal(T, hv, D) if norm else None}
    a_log, dt = torch.rand(hv, generator=gen, device=DEV), torch.randn(hv, generator=gen, device=DEV)
    w = 1 + 0.1 * torch.randn(D, generator=gen, device=DEV) if norm else None
    state = torch.randn(3, hv, D, D, generator=gen, device=DEV)
    kept, cu, at = state.clone(), ints([5, 40000, T - 3]), ints([2, 0])
    out = torch.full((T, hv, D), 7.0, device=DEV).bfloat16()
    la.linear_attn_prefill(q, k, v, x["g"], x["beta"], state, at, cu, qk_norm=True, a_log=a_log,
                           dt_bias=dt, z=x["z"], norm_weight=w, out=out)
    for h in (0, 29, 95, 96, 191):
        st, kh, one = kept[:, h:h + 1].contiguous(), h // 96, slice(h, h + 1)
        some = {n: None if t is None else t[:, one].contiguous() for n, t in x.items()}
        want = la.linear_attn_prefill(q[:, kh:kh + 1].contiguous(), k[:, kh:kh + 1].contiguous(),
                                      v[:, one].contiguous(), some["g"], some["beta"], st, at, cu,
                                      qk_norm=True, a_log=a_log[one], dt_bias=dt[one], z=some["z"],
                                      norm_weight=w)
        rows = slice(5, T - 3)
        for got, ref_, tol in ((out[rows, one], want[rows], 2.0 ** -7), (state[:, one], st, 1e-5)):
            ref_ = ref_.double()
            assert (got.double() - ref_).norm() <= tol * ref_.norm(), h
    la.check_errors(DEV)
    assert (out[:5] == 7).all() and (out[T - 3:] == 7).all() and torch.equal(state[1], kept[1])
