"""The paged cache's operators on the GPU against plain implementations: the
plan against a simulation in Python, the codec and the sketch against the
oracle, norm with rotation and attention against 64-bit numpy; at the sizes,
strides, tables and lengths where they can go wrong, and run together."""
import math

import numpy as np
import pytest

from oracle import oracle as orc

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ALL = orc.OUTLIER_ALL


@pytest.fixture(scope="module")
def tq():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import turboquant_amd
    return turboquant_amd


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ---------------------------------------------------------------- plan

def simulate(kv, new, table, free, count, page, tokens):
    """One step on the host; table and free are written."""
    kv, free_n = [int(x) for x in kv], int(count)
    width, batch = table.shape[1], len(kv)
    pages = lambda t: min(-(-t // page), width)  # noqa: E731
    for b in range(batch):
        if new[b] < 0:
            for j in range(pages(max(kv[b], 0))):
                free[free_n] = table[b, j]
                free_n += 1
    slots, pos = np.full(tokens, -1, np.int64), np.full(tokens, -1, np.int32)
    starts, appended, out = [0], [], []
    wanted = taken = 0
    for b in range(batch):
        n, start = max(int(new[b]), 0), starts[-1]
        starts.append(start + n)
        room = kv[b] + n <= width * page and start + n <= tokens
        held = pages(kv[b])
        need = pages(kv[b] + n) - held if room else 0
        wanted += need
        fits = room and (need == 0 or wanted <= free_n)
        appended.append(n if fits else 0)
        out.append(0 if new[b] < 0 else kv[b] + (n if fits else 0))
        if not fits:
            continue
        for j in range(need):
            table[b, held + j] = free[free_n - 1 - (wanted - need) - j]
        taken += need
        for i in range(n):
            p = kv[b] + i
            slots[start + i], pos[start + i] = int(table[b, p // page]) * page + p % page, p
    return slots, pos, np.array(starts), np.array(appended), np.array(out), free_n - taken


def plan_state(rng, batch, page, width, spare):
    """Random requests with their pages, and `spare` free pages; one request in ten fills its row."""
    kv = rng.integers(0, width * page + 1, size=batch).astype(np.int32)
    kv[rng.random(batch) < 0.1] = width * page
    held = -(-kv // page)
    ids = rng.permutation(int(held.sum()) + spare).astype(np.int32)
    table = np.full((batch, width), -7, np.int32)
    table[np.arange(width)[None] < held[:, None]] = ids[:held.sum()]
    free = np.concatenate((ids[held.sum():], np.full(int(held.sum()), -9, np.int32)))
    return kv, table, free


@pytest.mark.parametrize("batch,page,width,spare,most,tokens", [
    (1, 16, 1, 1, 1, 1), (1, 64, 8, 8, 300, 512), (5, 16, 40, 100, 200, 700), (64, 64, 20, 30, 1, 64),
    (64, 32, 10, 3, 1, 60), (300, 128, 6, 200, 5, 900), (1024, 16, 5, 900, 2, 1500), (1025, 16, 5, 2000, 3, 4000),
    (2500, 256, 3, 800, 40, 30000), (7, 1024, 30, 60, 9000, 60000), (33, 16, 2, 0, 1, 33), (3, 16, 4, 10, 2, 0)])
def test_plan_against_a_simulation(tq, batch, page, width, spare, most, tokens):
    rng = np.random.default_rng(batch * 7 + page)
    kv, table, free = plan_state(rng, batch, page, width, spare)
    new = np.where(rng.random(batch) < 0.2, -1, rng.integers(0, most + 1, size=batch)).astype(np.int32)
    new[rng.random(batch) < 0.1] = -2147483648
    tab, fr = dev(table), dev(free)
    args = (dev(kv), dev(new), tab, fr, i32(spare), page, tokens)
    p = tq.paged_plan(*args)
    slots, pos, starts, appended, out, left = simulate(kv, new, table, free, spare, page, tokens)
    for name, got, want in (("starts", p.starts, starts), ("appended", p.appended, appended), ("lens", p.kv_lens, out),
                            ("free", p.free_count, [left]), ("stack", fr, free), ("table", tab, table),
                            ("positions", p.positions, pos), ("slots", p.slots, slots)):
        assert np.array_equal(got.cpu().numpy(), np.asarray(want)), name
    # the same inputs again: the same step
    q = tq.paged_plan(*args)
    assert all(torch.equal(a, b) for a, b in zip(p, q))


def test_plan_in_place_over_steps(tq):
    """Lengths, table and free list carried on by the device, 30 steps of arrivals, growth and ends."""
    rng = np.random.default_rng(3)
    batch, page, width, pages = 40, 16, 12, 200
    kv, table = np.zeros(batch, np.int32), np.full((batch, width), -1, np.int32)
    free, count = np.arange(pages, dtype=np.int32), pages
    d = [dev(kv), dev(table), dev(free), i32(count)]
    for step in range(30):
        new = np.where(rng.random(batch) < 0.15, -1, rng.integers(0, 12, size=batch)).astype(np.int32)
        p = tq.paged_plan(d[0], dev(new), d[1], d[2], d[3], page, 250, kv_lens_out=d[0], free_count_out=d[3])
        slots, pos, _, _, kv, count = simulate(kv, new, table, free, count, page, 250)
        assert np.array_equal(p.slots.cpu().numpy(), slots) and np.array_equal(p.positions.cpu().numpy(), pos), step
        assert np.array_equal(d[0].cpu().numpy(), kv) and int(d[3]) == count, step
        assert np.array_equal(d[1].cpu().numpy(), table), step
        held = [table[b, j] for b in range(batch) for j in range(-(-int(kv[b]) // page))]
        assert sorted(held + list(free[:count])) == list(range(pages)), step  # every page has one owner


def test_plan_lengths_out_of_range(tq):
    """Negative lengths count as none; a request past its table row appends nothing; a free count past the list is cut."""
    table, free = dev(np.arange(6, dtype=np.int32).reshape(3, 2)), dev(np.arange(6, 10, dtype=np.int32))
    p = tq.paged_plan(i32(-5, 33, 32), i32(3, 1, 1), table, free, i32(99), 16, 8)
    assert p.appended.tolist() == [3, 0, 0] and p.kv_lens.tolist() == [3, 33, 32] and p.free_count.tolist() == [3]
    assert p.slots.tolist() == [9 * 16, 9 * 16 + 1, 9 * 16 + 2, -1, -1, -1, -1, -1]
    assert p.positions.tolist() == [0, 1, 2, -1, -1, -1, -1, -1] and table.tolist()[0] == [9, 1]
    n = 1 << 24  # the most that a step holds
    p = tq.paged_plan(i32(0), i32(n + 9), dev(np.zeros((1, 4), np.int32)), free, i32(4), 16, n)
    assert p.appended.tolist() == [0] and int(p.slots.max()) == -1
    p = tq.paged_plan(i32(0), i32((1 << 24) + 9), dev(np.zeros((1, 4), np.int32)), free, i32(4), 16, 4)
    assert p.appended.tolist() == [0] and p.slots.tolist() == [-1] * 4 and p.free_count.tolist() == [4]


# ---------------------------------------------------------------- norm and rotation

def rope_reference(x, pos, freq, w, eps, inter):
    y = x.astype(np.float64)
    if w is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * w
    n = len(freq)
    ang = pos.astype(np.float64)[:, None, None] * freq.astype(np.float64)
    c, s = np.cos(ang), np.sin(ang)
    one = np.arange(n) * 2 if inter else np.arange(n)
    two = one + 1 if inter else one + n
    a, b, out = y[..., one], y[..., two], y.copy()
    out[..., one], out[..., two] = a * c - b * s, b * c + a * s
    size = np.abs(y)
    size[..., one] = size[..., two] = np.abs(a) + np.abs(b)
    return out, size


def rope_bound(ref, size, dtype):
    """A chain of at most 20 f32 roundings of each term (the sum of squares counts half of its 13), each half a
    step, 2^-24; then half a step of the output, which for f16 is no smaller than half of 2^-24."""
    half = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}[dtype]
    return 20 * 2.0 ** -24 * size + half * np.abs(ref) + (2.0 ** -25 if dtype == "f16" else 1e-37)


def heads(rng, t, n, d, dtype):
    return dev(rng.standard_normal((t, n, d)).astype(np.float32) * 2).to(DT[dtype])


def as64(t):
    return t.float().cpu().numpy().astype(np.float64)


def check_rope(got, x, pos, freq, w, eps, inter, dtype):
    ref, size = rope_reference(as64(x), pos, freq, None if w is None else as64(w), eps, inter)
    err = np.abs(as64(got) - ref)
    assert (err <= rope_bound(ref, size, dtype)).all(), float((err / rope_bound(ref, size, dtype)).max())


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("d,rot", [(32, 32), (64, 64), (64, 32), (96, 96), (128, 128), (128, 64), (160, 40), (256, 256),
                                   (256, 64), (224, 224), (128, 6), (32, 2), (64, 0)])
@pytest.mark.parametrize("inter", [False, True])
def test_rope_shapes(tq, d, rot, inter, dtype):
    rng = np.random.default_rng(d + rot)
    t, hq, hk = 19, 5, 2
    q, k = heads(rng, t, hq, d, dtype), heads(rng, t, hk, d, dtype)
    pos = rng.integers(0, 40000, size=t).astype(np.int32)
    freq = (10000.0 ** (-np.arange(rot // 2) / max(1, rot // 2))).astype(np.float32)
    wq, wk = (dev(rng.random(d).astype(np.float32) + 0.5).to(DT[dtype]) for _ in range(2))
    qo, ko = tq.qk_norm_rope(q, k, dev(pos), dev(freq), wq, wk, 1e-5, inter)
    check_rope(qo, q, pos, freq, wq, 1e-5, inter, dtype)
    check_rope(ko, k, pos, freq, wk, 1e-5, inter, dtype)


@pytest.mark.parametrize("t", [1, 2, 63, 700])
@pytest.mark.parametrize("hq,hk", [(1, 1), (32, 8), (7, 1), (64, 64)])
def test_rope_tokens_and_heads(tq, t, hq, hk):
    rng = np.random.default_rng(t + hq)
    q, k = heads(rng, t, hq, 128, "bf16"), heads(rng, t, hk, 128, "bf16")
    pos = np.arange(t, dtype=np.int32) + 5
    freq = (1e6 ** (-np.arange(64) / 64)).astype(np.float32)
    w = dev(rng.random(128).astype(np.float32) + 0.5).to(torch.bfloat16)
    qo, ko = tq.qk_norm_rope(q, k, dev(pos), dev(freq), w, None)
    check_rope(qo, q, pos, freq, w, 1e-6, False, "bf16")
    check_rope(ko, k, pos, freq, None, 1e-6, False, "bf16")


@pytest.mark.parametrize("inter", [False, True])
def test_rope_far_positions(tq, inter):
    """Angles up to 2^31 rad: the f64 product's rounding, 2^-53 of the angle, is what the reference has too."""
    rng = np.random.default_rng(1)
    pos = np.array([0, 1, 1000003, 2 ** 24 + 1, 2 ** 31 - 1], np.int32)
    q, k = heads(rng, 5, 2, 64, "f32"), heads(rng, 5, 1, 64, "f32")
    freq = np.concatenate(([1.0, 0.5, 2.0, np.pi / 2, np.pi / 4], 10000.0 ** (-np.arange(27) / 27))).astype(np.float32)
    qo, ko = tq.qk_norm_rope(q, k, dev(pos), dev(freq), interleaved=inter)
    check_rope(qo, q, pos, freq, None, 0, inter, "f32")
    check_rope(ko, k, pos, freq, None, 0, inter, "f32")


@pytest.mark.parametrize("offset,extra", [(0, 0), (0, 40), (8, 24), (1, 3), (5, 8)])
@pytest.mark.parametrize("inter", [False, True])
def test_rope_strides_and_places(tq, offset, extra, inter):
    """Views of a projection's rows from any element on, in place, and rows of no token left as they were."""
    rng = np.random.default_rng(offset + extra)
    t, hq, hk, d = 33, 3, 2, 64
    width = (hq + 2 * hk) * d + extra
    buf = torch.zeros(t * width + offset, dtype=torch.float16, device="cuda")
    rows = buf[offset:].view(t, width)
    rows.copy_(dev(rng.standard_normal((t, width)).astype(np.float32)))
    q, k = rows[:, :hq * d].view(t, hq, d), rows[:, hq * d:(hq + hk) * d].view(t, hk, d)
    pos = np.arange(t, dtype=np.int32) * 17
    pos[[0, 4, 32]] = -1
    freq = (10000.0 ** (-np.arange(16) / 16)).astype(np.float32)
    w = dev(rng.random(d).astype(np.float32)).half()
    before, keep = rows.clone(), pos < 0
    qo, ko = tq.qk_norm_rope(q, k, dev(pos), dev(freq), w, w, interleaved=inter)
    check_rope(qo[~keep], q[~keep], pos[~keep], freq, w, 1e-6, inter, "f16")
    same = tq.qk_norm_rope(q, k, dev(pos), dev(freq), w, w, interleaved=inter, out=(q, k))
    assert same[0].data_ptr() == q.data_ptr()
    assert torch.equal(q[~keep], qo[~keep]) and torch.equal(k[~keep], ko[~keep])
    assert torch.equal(rows[keep], before[keep])                                  # no token: untouched
    assert torch.equal(rows[:, (hq + hk) * d:], before[:, (hq + hk) * d:])        # nor what lies behind
    with pytest.raises(ValueError, match="adjacent"):
        tq.qk_norm_rope(q[:, :, ::2], k[:, :, ::2], dev(pos), dev(freq[:8]))


def test_rope_zeros_infinities_and_nan(tq):
    q = torch.zeros(3, 2, 64, device="cuda")
    q[1, 0, 3], q[2, 1, 5] = float("inf"), float("nan")
    f = torch.ones(32, device="cuda")
    qo, _ = tq.qk_norm_rope(q, q, i32(0, 1, 2), f, torch.ones(64, device="cuda"))
    assert (qo[0] == 0).all() and (qo[1, 1] == 0).all() and (qo[2, 0] == 0).all()
    assert qo[1, 0].isnan().any() and qo[2, 1].isnan().all()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("d,rot", [(64, 32), (128, 6), (96, 64), (64, 0)])
@pytest.mark.parametrize("inter", [False, True])
def test_rope_passes_the_rest_of_a_head_through(tq, d, rot, inter, dtype):
    """Without a norm the elements past rot_dim come out as they are, infinities and what stands beside them too."""
    rng = np.random.default_rng(d + rot)
    q = heads(rng, 5, 3, d, dtype)
    q[:, 0, rot], q[:, 1, d - 1], q[2, 2, rot + 5] = float("inf"), float("-inf"), float("inf")
    freq = dev((10000.0 ** (-np.arange(rot // 2) / max(1, rot // 2))).astype(np.float32))
    qo, ko = tq.qk_norm_rope(q, q[:, :2], i32(0, 1, 7, 500, 30000), freq, interleaved=inter)
    assert torch.equal(qo[..., rot:], q[..., rot:]) and torch.equal(ko, qo[:, :2])
    assert qo[..., :rot].isfinite().all()


def test_wrappers_refuse(tq):
    """Shapes, types, strides and places that the wrappers check themselves."""
    q, k, pos, f = torch.zeros(3, 4, 64).cuda(), torch.zeros(3, 2, 64).cuda(), i32(0, 1, 2), torch.ones(32).cuda()
    layer = tq.PagedLayer.empty(2, 16, 2, 64, 3)
    slots, ws = torch.arange(3).cuda(), tq.AttentionWorkspace(3, 4, 2, 64, 32)
    table = torch.zeros((3, 2), dtype=torch.int32, device="cuda")
    for call in (lambda: tq.qk_norm_rope(q, k, pos, f, out=(k, k)), lambda: tq.qk_norm_rope(q, k, pos.long(), f),
                 lambda: tq.qk_norm_rope(q, k, pos, f.double()), lambda: tq.qk_norm_rope(q, k, pos, f, q[0, 0, :32]),
                 lambda: tq.qk_norm_rope(q, k, pos, f, q[0, 0].half()), lambda: tq.qk_norm_rope(q, k, pos[:2], f),
                 lambda: tq.qk_norm_rope(q, k, pos.cpu(), f), lambda: tq.qk_norm_rope(q.transpose(0, 1), k, pos, f),
                 lambda: tq.paged_store(layer, slots, k, k, 4), lambda: tq.paged_store(layer, slots, k, k.half(), 3),
                 lambda: tq.paged_store(layer, slots.int(), k, k, 3), lambda: tq.paged_store(layer, slots, q, q, 3),
                 lambda: tq.paged_store(layer, slots, k, k, 3, 0, sign_matrix=f),
                 lambda: tq.paged_load(layer, slots, 3, out=(k, k.half())),
                 lambda: tq.paged_load(layer, slots[::2], 3, out=(k[:2], k[:2])),
                 lambda: tq.paged_decode_attention(q[:, :, :32], layer, table, pos, 3, 32, 1.0, ws),
                 lambda: tq.paged_decode_attention(q, layer, table, pos.long(), 3, 32, 1.0, ws),
                 lambda: tq.paged_decode_attention(q, layer, table[:2], pos, 3, 32, 1.0, ws),
                 lambda: tq.paged_decode_attention(q, layer, table, pos, 3, 32, 1.0, ws, sign_matrix=f.int()),
                 lambda: tq.paged_plan(pos, pos, table, pos[::2], pos[:1], 16, 3),
                 lambda: tq.paged_plan(pos, pos[:2], table, pos, pos[:1], 16, 3),
                 lambda: tq.paged_plan(pos, pos, table, pos, pos[:1], 16, -1)):
        with pytest.raises(ValueError):
            call()
    cache = tq.PagedCache(tq.CacheConfig(3, 64, 2, 1), 4, 3, 32, 16)
    plan = cache.plan(i32(1, 1, 1), 3)
    for call in (lambda: cache.step(0, plan, q[:2], k, k, 1.0), lambda: cache.step(0, plan, q[:0], k[:0], k[:0], 1.0),
                 lambda: cache.attend(0, q[:2], 1.0)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(tq.TurboQuantError, match="exceeds a table row"):
        tq.paged_decode_attention(q, layer, table, pos, 3, 33, 1.0, ws)


# ---------------------------------------------------------------- records in pages

def layer_and_slots(tq, rng, t, page, hk, d, bits, qjl, spare=2):
    pages = -(-t // page) + spare
    layer = tq.PagedLayer.empty(pages, page, hk, d, bits, qjl)
    order = rng.permutation(pages)
    at = np.arange(t) + (3 if t + 3 <= pages * page else 0)
    return layer, (order[at // page] * page + at % page).astype(np.int64)


def at(pool, slots, page):
    """Records [t, heads, ...] of slots in a pool."""
    s = torch.from_numpy(slots).cuda()
    return pool[s // page, :, s % page].cpu().numpy()


@pytest.mark.parametrize("t,page,hk,d,bits,ob,norm,dtype", [
    (1, 16, 1, 32, 3, ALL, 0, "f32"), (40, 16, 2, 128, 3, ALL, 0, "bf16"), (17, 64, 8, 128, 4, ALL, 0, "f16"),
    (300, 32, 3, 64, 3, 0, 0, "bf16"), (129, 128, 2, 256, 4, 0, 0, "f32"), (77, 16, 2, 96, 4, ALL, 0, "bf16"),
    (50, 256, 1, 128, 3, ALL, 1, "f32"), (50, 1024, 2, 64, 4, 0, 1, "bf16"), (9, 16, 5, 160, 3, ALL, 0, "f16")])
def test_store_and_load(tq, t, page, hk, d, bits, ob, norm, dtype):
    rng = np.random.default_rng(t + d)
    layer, slots = layer_and_slots(tq, rng, t, page, hk, d, bits, False)
    both = (dev(rng.standard_normal((t, 2 * hk, d)).astype(np.float32)) * 3).to(DT[dtype])
    k, v = both[:, :hk], both[:, hk:]  # rows 2 hk d apart
    with_pad = slots.copy()
    with_pad[::5] = [-1, layer.num_pages * page, -2 ** 62, 2 ** 62][t % 4]  # rows of no token
    live = np.arange(t) % 5 != 0
    tq.paged_store(layer, dev(with_pad), k, v, bits, ob, norm)
    ko = torch.full((t, hk, d), 7.0, device="cuda").to(DT[dtype])
    vo = ko.clone()
    tq.paged_load(layer, dev(with_pad), bits, ob, norm, out=(ko, vo))
    for x, idx, sc, back in ((k, layer.k_idx, layer.k_sc, ko), (v, layer.v_idx, layer.v_sc, vo)):
        p, s = orc.polar_quantize(bits, ob, x.float().cpu().numpy().reshape(-1, d), d, norm)
        assert np.array_equal(at(idx, slots, page)[live], p.reshape(t, hk, -1)[live])
        assert np.array_equal(at(sc, slots, page)[live].view(np.uint16), s.reshape(t, hk, -1)[live])
        assert not at(idx, slots, page)[~live].any()
        ref = torch.from_numpy(orc.polar_dequantize(bits, ob, p, s, d, norm)).view(t, hk, d).to(DT[dtype])
        assert torch.equal(back.cpu()[live], ref[live]) and (back.cpu()[~live] == 7).all()
        written = int(live.sum()) * hk
        assert int((sc != 0).any(-1).sum()) <= written  # nothing beside the slots
    one = tq.paged_load(layer, dev(slots[live]), bits, ob, norm, torch.float32)
    assert torch.equal(one[0].to(DT[dtype]), ko[torch.from_numpy(live).cuda()])


def test_store_from_any_element(tq):
    """k and v off the 16-byte boundary, and at odd strides."""
    rng = np.random.default_rng(5)
    t, page, hk, d, bits = 21, 16, 2, 64, 3
    layer, slots = layer_and_slots(tq, rng, t, page, hk, d, bits, False)
    buf = dev(rng.standard_normal(t * 131 * 2 + 1).astype(np.float32)).to(torch.bfloat16)
    k = buf[1:1 + t * 131].view(t, 131)[:, :128].view(t, hk, d)
    v = buf[1 + t * 131:].view(t, 131)[:, 3:].view(t, hk, d)
    tq.paged_store(layer, dev(slots), k, v, bits)
    for x, idx in ((k, layer.k_idx), (v, layer.v_idx)):
        p, _ = orc.polar_quantize(bits, ALL, x.float().cpu().numpy().reshape(-1, d), d)
        assert np.array_equal(at(idx, slots, page), p.reshape(t, hk, -1))


@pytest.mark.parametrize("t,page,hk,d,bits,norm,dtype", [
    (1, 16, 1, 64, 3, 0, "f32"), (40, 16, 3, 128, 3, 0, "bf16"), (33, 64, 2, 128, 4, 0, "f16"),
    (130, 32, 1, 256, 4, 0, "bf16"), (20, 16, 2, 256, 3, 1, "f32"), (47, 128, 2, 64, 4, 1, "bf16")])
def test_store_tq(tq, t, page, hk, d, bits, norm, dtype):
    rng = np.random.default_rng(t + d)
    layer, slots = layer_and_slots(tq, rng, t, page, hk, d, bits, True)
    k, v = ((dev(rng.standard_normal((t, hk, d)).astype(np.float32)) * 2).to(DT[dtype]) for _ in range(2))
    with_pad = slots.copy()
    with_pad[1::4] = -1
    live = with_pad >= 0
    rmat = tq.qjl_sign_matrix(d, 12345)
    tq.paged_store(layer, dev(with_pad), k, v, bits, 0, norm, sign_matrix=rmat)
    for x, idx, sc in ((k, layer.k_idx, layer.k_sc), (v, layer.v_idx, layer.v_sc)):
        xs = x.float().cpu().numpy().reshape(-1, d)
        p, s = orc.polar_quantize(bits, 0, xs, d, norm)
        assert np.array_equal(at(idx, slots, page)[live], p.reshape(t, hk, -1)[live])
        assert np.array_equal(at(sc, slots, page)[live].view(np.uint16), s.reshape(t, hk, -1)[live])
        if x is k:
            sg, nm = orc.tq_signs_norms(xs, orc.polar_dequantize(bits, 0, p, s, d, norm))
            assert np.array_equal(at(layer.signs, slots, page)[live], sg.reshape(t, hk, -1)[live])
            assert np.array_equal(at(layer.norms, slots, page)[live].view(np.uint16), nm.reshape(t, hk)[live])
    assert not at(layer.signs, slots, page)[~live].any() and not at(layer.norms, slots, page)[~live].any()


# ---------------------------------------------------------------- attention

def filled(tq, rng, lens, page, width, hk, d, bits, mode):
    """A layer whose requests' pages hold random tokens, with garbage behind them and in every other page; the table
    (entries behind a request's pages wild); and the requests' keys, values and logit correction operands."""
    pages = sum(-(-n // page) for n in lens) + 3
    layer = tq.PagedLayer.empty(pages, page, hk, d, bits, mode == "tq")
    for pool in (layer.k_idx, layer.v_idx):
        pool.random_(0, 256)
    for pool in (layer.k_sc, layer.v_sc):
        pool.fill_(0x7e00)  # NaN
    if mode == "tq":
        layer.signs.random_(0, 256)
        layer.norms.fill_(0x7c00)  # infinity
    order = rng.permutation(pages)
    table = rng.integers(-2 ** 31, 2 ** 31, size=(len(lens), width)).astype(np.int32)
    ob = ALL if mode == "pqo" else 0
    rmat = tq.qjl_sign_matrix(d, 12345) if mode == "tq" else None
    used, recs = 0, []
    for b, n in enumerate(lens):
        own = -(-n // page)
        table[b, :own] = order[used:used + own]
        used += own
        x = [rng.standard_normal((n, hk, d)).astype(np.float32) for _ in range(2)]
        x[0][..., rng.choice(d, 2)] *= 5
        if n:
            at_ = np.arange(n)
            slots = table[b, at_ // page].astype(np.int64) * page + at_ % page
            k, v = (dev(a) for a in x)
            tq.paged_store(layer, dev(slots), k, v, bits, ob, sign_matrix=rmat)
            k, v = (as64(a) for a in tq.paged_load(layer, dev(slots), bits, ob))
            sg = np.unpackbits(at(layer.signs, slots, page), axis=-1, bitorder="little") * 2.0 - 1 if rmat is not None else None
            nm = at(layer.norms, slots, page).view(np.float16).astype(np.float64) if rmat is not None else None
            recs.append((k, v, sg, nm))
        else:
            recs.append(None)
    return layer, dev(table), ob, rmat, recs


def sign_rows(rmat, d):
    w = rmat.cpu().numpy().view(np.uint32).reshape(d, d // 32)
    return 1.0 - 2.0 * ((w[:, :, None] >> np.arange(32)) & 1).reshape(d, d)


def attend(q, recs, scale, rmat, skip=None, codebook=0.0):
    """64-bit attention of q [H, D] over a request's records, and a bound of a kernel's error: logits of two-part f16
    operands are off by 2^-20 of the sum of their terms' sizes (twice that where a correction joins), weights by as
    much twice (numerator and sum), and values, whose products are cut likewise and whose offset grows them by up to
    2 x 2.16 x sqrt(32), by 2^-16 of the largest.  `codebook`: centroids off by as much of their size, so logits by as
    much of their terms', and a value, 32 centroids in an orthogonal transform, by sqrt(32) times as much of the
    largest."""
    h, d = q.shape
    out, bound = np.zeros((h, d)), np.zeros((h, 1))
    if recs is None:
        return out, bound
    k, v, sg, nm = recs
    keep = np.ones(len(k), bool) if skip is None else ~skip
    if not keep.any():
        return out, bound
    k, v = k[keep], v[keep]
    for i in range(h):
        g = i // (h // k.shape[1])
        x, size = k[:, g] @ q[i], np.abs(k[:, g]) @ np.abs(q[i])
        if rmat is not None:
            rq = sign_rows(rmat, d) @ q[i] / math.sqrt(d)
            c = nm[keep][:, g] * math.sqrt(math.pi / 2) / math.sqrt(d)
            x, size = x + (sg[keep][:, g] @ rq) * c, size + np.abs(rq).sum() * c
        w = np.exp((x - x.max()) * scale)
        out[i] = w @ v[:, g] / w.sum()
        top = np.abs(v[:, g]).max()
        bound[i] = top * (4 * scale * (2.0 ** -20 + codebook) * size.max() + 2.0 ** -16 + codebook * math.sqrt(32))
    return out, bound


def half_step(ref, dtype):
    return np.abs(ref) * {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}[dtype] + 2.0 ** -25


def check_attention(tq, lens, page, width, hq, hk, d, bits, mode, dtype="bf16", out="f32", most=None, seed=0):
    rng = np.random.default_rng(seed + sum(lens) + d + hq)
    layer, table, ob, rmat, recs = filled(tq, rng, lens, page, width, hk, d, bits, mode)
    q = dev(rng.standard_normal((len(lens), hq, d)).astype(np.float32)).to(DT[dtype])
    most = width * page if most is None else most
    ws = tq.AttentionWorkspace(len(lens), hq, hk, d, most)
    got = tq.paged_decode_attention(q, layer, table, i32(*lens), bits, most, d ** -0.5, ws, ob, sign_matrix=rmat,
                                    out_dtype=DT[out])
    # 16-bit results of 3-bit codes may come from a codebook rounded to f16 at its best scale
    codebook = 2.0 ** -15.4 if bits == 3 and out != "f32" else 0.0
    for b in range(len(lens)):
        ref, bound = attend(as64(q[b]), recs[b], d ** -0.5, rmat, codebook=codebook)
        err = np.abs(as64(got[b]) - ref)
        assert (err <= bound + half_step(ref, out)).all(), (b, lens[b], float(err.max()), float(bound.max()))
    return q, layer, table, ob, rmat, recs, ws


@pytest.mark.parametrize("mode,bits", [("pqo", 3), ("pqo", 4), ("pq", 3), ("pq", 4), ("tq", 3), ("tq", 4)])
@pytest.mark.parametrize("d", [32, 64, 128, 256])
def test_decode_modes_and_dims(tq, mode, bits, d):
    if mode == "tq" and d == 32:
        pytest.skip("no sketch of 32 elements")
    check_attention(tq, [700, 1, 16, 333], 32, 24, 4, 2, d, bits, mode)


@pytest.mark.parametrize("hq,hk", [(1, 1), (2, 1), (3, 1), (8, 1), (16, 1), (12, 4), (5, 5), (20, 2)])
@pytest.mark.parametrize("mode,bits", [("pqo", 3), ("pqo", 4), ("tq", 3)])
def test_decode_heads(tq, hq, hk, mode, bits):
    check_attention(tq, [130, 515], 16, 40, hq, hk, 64, bits, mode)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256, 1024])
@pytest.mark.parametrize("mode,bits", [("pqo", 3), ("pqo", 4), ("tq", 4)])
def test_decode_pages_and_lengths(tq, page, mode, bits):
    lens = [0, 1, 15, 16, 17, page - 1, page, page + 1, 2 * page, 3 * page + 7, 511, 512, 513, 1025, 2100]
    check_attention(tq, lens, page, -(-2100 // page) + 1, 4, 2, 128, bits, mode)


@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f16", "bf16")])
@pytest.mark.parametrize("mode,bits", [("pqo", 3), ("pqo", 4), ("tq", 3)])
def test_decode_types(tq, dtype, out, mode, bits):
    check_attention(tq, [90, 1300], 64, 21, 8, 2, 128, bits, mode, dtype, out)


@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("mode,bits", [("pqo", 3), ("pqo", 4), ("pq", 3), ("pq", 4), ("tq", 3), ("tq", 4)])
def test_decode_long(tq, mode, bits, out):
    """Contexts split over many workgroups, joined, beside short ones."""
    check_attention(tq, [20001, 37, 9000], 64, 320, 4, 2, 128, bits, mode, out=out)


@pytest.mark.parametrize("batch,hk,group,out", [(70, 8, 1, "f32"), (200, 2, 1, "bf16"), (300, 1, 1, "f32"),
                                                (300, 1, 2, "f16"), (64, 16, 1, "f16"), (40, 40, 1, "f32"),
                                                (64, 8, 4, "f16"), (90, 8, 2, "bf16"), (20, 40, 1, "f16"),
                                                (40, 4, 16, "f16"), (256, 4, 1, "f16"), (257, 4, 1, "f16")])
@pytest.mark.parametrize("mode,bits", [("pqo", 3), ("pqo", 4), ("tq", 3)])
def test_decode_many_requests(tq, batch, hk, group, out, mode, bits):
    """About and more (request, KV head) pairs than workgroups are resident at once, some of them empty."""
    rng = np.random.default_rng(batch)
    lens = rng.integers(0, 900, size=batch).tolist()
    lens[3], lens[-1] = 0, 1800
    check_attention(tq, lens, 64, 29, hk * group, hk, 64, bits, mode, out=out)


@pytest.mark.parametrize("d,group", [(32, 1), (32, 8), (128, 1), (128, 4), (128, 8), (256, 2), (256, 8)])
@pytest.mark.parametrize("mode,bits", [("pqo", 3), ("pq", 3), ("tq", 3), ("pqo", 4)])
def test_decode_range_launches(tq, d, group, mode, bits):
    """16-bit results of batches that take ranges of several chunks, at every shape of head; pages from tile to chunk."""
    if mode == "tq" and d == 32:
        pytest.skip("no sketch of 32 elements")
    lens = [5000, 1, 128, 127, 129, 513, 2047, 4096, 0, 3333, 511, 1025] * 2
    check_attention(tq, lens, 16 if group == 1 else 256, 320 if group == 1 else 20, 8 * group, 8, d, bits, mode, out="f16")


def test_decode_lengths_are_clamped(tq):
    """Negative lengths are none; those past max_kv_len end there."""
    rng = np.random.default_rng(0)
    layer, table, ob, _, recs = filled(tq, rng, [100, 100, 100], 16, 8, 1, 64, 3, "pqo")
    q = dev(rng.standard_normal((3, 2, 64)).astype(np.float32))
    ws = tq.AttentionWorkspace(3, 2, 1, 64, 70)
    got = tq.paged_decode_attention(q, layer, table, i32(-4, 2 ** 31 - 1, 60), 3, 70, 0.125, ws)
    assert (got[0] == 0).all()
    for b, n in ((1, 70), (2, 60)):
        ref, bound = attend(as64(q[b]), tuple(None if a is None else a[:n] for a in recs[b]), 0.125, None)
        assert (np.abs(as64(got[b]) - ref) <= bound + half_step(ref, "f32")).all()


@pytest.mark.parametrize("mode,bits", [("pqo", 3), ("pqo", 4), ("tq", 3)])
def test_decode_skips_entries_outside_the_pages(tq, mode, bits):
    """Table entries outside [0, num_pages) hold no tokens: in the middle, everywhere."""
    lens = [600, 600, 2600]
    q, layer, table, ob, rmat, recs, ws = check_attention(tq, lens, 64, 41, 4, 2, 128, bits, mode)
    bad = table.clone()
    bad[0, 2], bad[0, 9], bad[1, :] = layer.num_pages, -1, -1
    bad[2, 10:31] = 2 ** 31 - 1
    got = tq.paged_decode_attention(q, layer, bad, i32(*lens), bits, 41 * 64, 128 ** -0.5, ws, ob, sign_matrix=rmat,
                                    out_dtype=torch.float32)
    assert (got[1] == 0).all()
    for b in (0, 2):
        p = np.arange(lens[b]) // 64
        skip = np.isin(p, [2, 9]) if b == 0 else (p >= 10) & (p < 31)
        ref, bound = attend(as64(q[b]), recs[b], 128 ** -0.5, rmat, skip)
        assert (np.abs(as64(got[b]) - ref) <= bound + half_step(ref, "f32")).all(), b


def test_decode_two_requests_share_pages(tq):
    """A common prefix: both rows name the same pages, and one request twice."""
    q, layer, table, ob, rmat, recs, _ = check_attention(tq, [500, 320], 64, 8, 4, 2, 128, 3, "pqo")
    t = torch.stack((table[0], table[0], table[0]))
    q3 = torch.stack((q[0], q[0], q[1]))
    ws = tq.AttentionWorkspace(3, 4, 2, 128, 512)
    got = tq.paged_decode_attention(q3, layer, t, i32(500, 500, 129), 3, 512, 128 ** -0.5, ws, out_dtype=torch.float32)
    assert torch.equal(got[0], got[1])
    ref, bound = attend(as64(q[1]), tuple(None if a is None else a[:129] for a in recs[0]), 128 ** -0.5, None)
    assert (np.abs(as64(got[2]) - ref) <= bound + half_step(ref, "f32")).all()


def test_decode_more_than_4_gib_of_pages(tq):
    """A page whose records begin past 2^32 bytes of the pool."""
    page, hk, d, bits = 1024, 8, 128, 4
    pages = (1 << 32) // (page * hk * 64) + 3
    layer = tq.PagedLayer.empty(pages, page, hk, d, bits)
    n, own = 1500, [pages - 1, pages - 2]
    rng = np.random.default_rng(0)
    at_ = np.arange(n)
    slots = dev(np.array(own)[at_ // page].astype(np.int64) * page + at_ % page)
    k, v = (dev(rng.standard_normal((n, hk, d)).astype(np.float32)) for _ in range(2))
    tq.paged_store(layer, slots, k, v, bits)
    k, v = (as64(a) for a in tq.paged_load(layer, slots, bits))
    assert np.abs(k).max() > 1
    q = dev(rng.standard_normal((1, hk, d)).astype(np.float32))
    ws = tq.AttentionWorkspace(1, hk, hk, d, 2048)
    got = tq.paged_decode_attention(q, layer, i32(*own)[None].contiguous(), i32(n), bits, 2048, d ** -0.5, ws)
    ref, bound = attend(as64(q[0]), (k, v, None, None), d ** -0.5, None)
    assert (np.abs(as64(got[0]) - ref) <= bound + half_step(ref, "f32")).all()


@pytest.mark.parametrize("mode", ["pqo", "tq"])
def test_decode_repeats_bit_for_bit(tq, mode):
    q, layer, table, ob, rmat, _, ws = check_attention(tq, [5000, 4, 811], 64, 80, 8, 4, 128, 3, mode)
    args = (q, layer, table, i32(5000, 4, 811), 3, 5120, 128 ** -0.5, ws, ob)
    first = tq.paged_decode_attention(*args, sign_matrix=rmat)
    for _ in range(5):
        assert torch.equal(tq.paged_decode_attention(*args, sign_matrix=rmat), first)


# ---------------------------------------------------------------- together

def rope_of(tq, d):
    freq = (10000.0 ** (-np.arange(d // 2) / (d // 2))).astype(np.float32)
    w = torch.linspace(0.6, 1.4, d, device="cuda").to(torch.bfloat16)
    return tq.QkNormRope(dev(freq), w, w)


@pytest.mark.parametrize("mode,bits,d", [("pqo", 3, 128), ("pqo", 4, 64), ("tq", 3, 128)])
def test_serving_steps_against_contiguous_caches(tq, mode, bits, d):
    """Prompts, then decode steps of a batch in which a request ends and another takes its place, against a
    contiguous cache per request fed with the same normed and rotated heads."""
    rng = np.random.default_rng(bits)
    hq, hk, layers, requests = 8, 2, 2, 3
    config = tq.CacheConfig(bits=bits, head_dim=d, num_kv_heads=hk, num_layers=layers,
                            outlier_blocks=tq.cache.OUTLIER_ALL if mode == "pqo" else 0)
    cache = tq.PagedCache(config, 40, requests, 300, page_size=16, qjl=mode == "tq")
    rope, scale = rope_of(tq, d), d ** -0.5
    make = lambda: (tq.TqCache if mode == "tq" else tq.PqoCache)(config)  # noqa: E731
    plain, length = [make() for _ in range(requests)], [0] * requests
    cfg = tq.AttendConfig(scale, hq // hk)

    def rows(t):
        x = dev(rng.standard_normal((t, hq + 2 * hk, d)).astype(np.float32)).to(torch.bfloat16)
        return x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]

    def step(new, pad):
        starts = np.concatenate(([0], np.cumsum(np.maximum(new, 0))))
        plan = cache.plan(i32(*new), int(starts[-1]) + pad)
        for b, n in enumerate(new):
            if n < 0:
                plain[b], length[b] = make(), 0
        for layer in range(layers):
            q, k, v = rows(int(starts[-1]) + pad)
            if max(new) > 1:
                q, k = tq.qk_norm_rope(q, k, plan.positions, *rope)
                cache.store(layer, plan, k, v)
                out = None
            else:
                out = cache.step(layer, plan, q, k, v, scale, rope)
                q, k = tq.qk_norm_rope(q, k, plan.positions, *rope)
            for b, n in enumerate(new):
                if n <= 0:
                    continue
                part = [x[starts[b]:starts[b + 1]].transpose(0, 1)[None].contiguous() for x in (k, v, q)]
                if out is None:
                    plain[b].prefill(layer, *part) if mode == "tq" else plain[b].prefill(layer, *part[:2])
                    continue
                ref = plain[b].decode(layer, *part, cfg)
                # the same records attended by two launches of this library: each within a bf16 step of the other
                assert (out[b].float() - ref[0, :, 0].float()).abs().max() <= 2.0 ** -7 * ref.float().abs().max(), (b, layer)
        for b, n in enumerate(new):
            length[b] += max(n, 0)
        assert cache.kv_lens.tolist() == length

    step([37, 5, 100], 3)
    for _ in range(4):
        step([1, 1, 1], 0)
    step([1, -1, 0], 2)
    step([0, 20, 0], 0)
    for _ in range(3):
        step([1, 1, 1], 1)
    owned = sum(-(-n // 16) for n in length)
    assert int(cache.free_count) == 40 - owned


def test_a_captured_step_replays(tq):
    """Plan, norm with rotation, store and attention captured once and replayed as requests grow over page borders,
    with eager work in between, against the same steps run eagerly."""
    d, hq, hk, requests = 128, 8, 2, 4
    config = tq.CacheConfig(bits=3, head_dim=d, num_kv_heads=hk, num_layers=1)
    rope = rope_of(tq, d)
    x = torch.empty(requests, hq + 2 * hk, d, dtype=torch.bfloat16, device="cuda")
    new = torch.ones(requests, dtype=torch.int32, device="cuda")

    def one(cache):
        plan = cache.plan(new, requests)
        return cache.step(0, plan, x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:], d ** -0.5, rope), plan.slots

    def prompt(cache):
        g = torch.Generator(device="cuda").manual_seed(1)
        plan = cache.plan(i32(14, 1, 700, 0), 800)
        k, v = (torch.randn(800, hk, d, device="cuda", generator=g).to(torch.bfloat16) for _ in range(2))
        cache.store(0, plan, k, v)

    caches = [tq.PagedCache(config, 80, requests, 1024, page_size=16) for _ in range(2)]
    for c in caches:
        prompt(c)
        c.attend(0, torch.zeros(requests, hq, d, dtype=torch.bfloat16, device="cuda"), 1.0)  # its workspace
    lens = [c.kv_lens.clone() for c in caches]
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    x.normal_()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        out, slots = one(caches[1])
    torch.cuda.synchronize()
    assert torch.equal(caches[1].kv_lens, lens[1])  # captured, not run
    g = torch.Generator(device="cuda").manual_seed(2)
    for i in range(20):
        x.copy_(torch.randn(x.shape, device="cuda", generator=g))
        ref, ref_slots = one(caches[0])
        graph.replay()
        assert torch.equal(ref_slots, slots), i
        assert torch.equal(ref, out), i
        assert caches[0].kv_lens.tolist() == caches[1].kv_lens.tolist()


def test_a_workspace_is_made_outside_of_a_capture_and_stays(tq, monkeypatch):
    """A graph's workspace is not given back when another number of heads asks for its own."""
    cache = tq.PagedCache(tq.CacheConfig(3, 64, 2, 1), 64, 2, 512, 16)
    k = torch.randn(700, 2, 64, device="cuda")
    cache.store(0, cache.plan(i32(450, 250), 700), k, k.flip(0))
    few, many = torch.randn(2, 4, 64, device="cuda"), torch.randn(2, 16, 64, device="cuda")
    with monkeypatch.context() as m:
        m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        with pytest.raises(RuntimeError, match="before the capture"):
            cache.attend(0, few, 0.125)
    ref = cache.attend(0, few, 0.125)
    held = cache._ws[4].buf.data_ptr()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        out = cache.attend(0, few, 0.125)
    for _ in range(3):
        other = cache.attend(0, many, 0.125)
        graph.replay()
        assert torch.equal(out, ref) and cache._ws[4].buf.data_ptr() == held
        assert torch.equal(other, cache.attend(0, many, 0.125))


def test_on_another_stream(tq):
    """The calls run on the current stream: work that it waits for is seen."""
    d, hk, n = 64, 1, 300
    layer = tq.PagedLayer.empty(30, 16, hk, d, 3)
    side = torch.cuda.Stream()
    k = torch.zeros(n, hk, d, device="cuda")
    slots = torch.arange(n, device="cuda")
    table, lens = torch.arange(20, dtype=torch.int32, device="cuda")[None], i32(n)
    q = torch.ones(1, 2, d, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        k.fill_(1.5)
        tq.paged_store(layer, slots, k, k, 3)
        ws = tq.AttentionWorkspace(1, 2, hk, d, 320)
        out = tq.paged_decode_attention(q, layer, table, lens, 3, 320, 0.125, ws)
        kk, _ = tq.paged_load(layer, slots, 3)
    side.synchronize()
    record = orc.polar_dequantize(3, ALL, *orc.polar_quantize(3, ALL, np.full((1, d), 1.5, np.float32), d), d)
    assert np.array_equal(kk.cpu().numpy(), np.broadcast_to(record, (n, hk, d)))
    # all values alike: their weighted sum is off by the bound of `attend` alone
    assert np.abs(as64(out) - record.astype(np.float64)).max() <= 2.0 ** -15 * np.abs(record).max()
