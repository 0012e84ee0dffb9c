"""The pool of resident scenes: block tables, slot maps and moved rows against their sequential definitions, and the whole way
from an augmented batch to the gradients of a training step."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def tables_by_rows(lengths, block, tables, held, free, n_free):
    """The definition, row after row."""
    tables, held = [list(r) for r in tables], list(held)
    stack = list(free[:n_free])
    blocks, most = len(free), len(tables[0])
    status = 0
    have = [min(most, -(-h // block)) if h > 0 else 0 for h in held]
    need = []
    for i, n in enumerate(lengths):
        k = -(-n // block) if n > 0 else 0
        fits = n >= 0 and k <= most
        need.append(k if fits else have[i])
        status |= not fits
    for i in range(len(tables)):
        if need[i] < have[i]:
            stack += tables[i][need[i]:have[i]]
            tables[i][need[i]:] = [-1] * (most - need[i])
    out = False
    for i in range(len(tables)):
        grow = need[i] - have[i]
        out = out or (grow > len(stack))
        if grow > 0 and out:
            status = 1
            continue
        for c in range(have[i], have[i] + max(0, grow)):
            tables[i][c] = stack.pop()
        n = lengths[i]
        if n >= 0 and -(-n // block) <= most:
            held[i] = n
    for i in range(len(tables)):
        k = -(-held[i] // block) if held[i] > 0 else 0
        tables[i][k:] = [-1] * (most - k)
    return tables, held, stack + [-1] * (blocks - len(stack)), len(stack), 16 if status else 0


def i32(v):
    return torch.tensor(np.asarray(v, dtype=np.int32)).cuda()


@pytest.mark.parametrize("rows,most,block,spare", [(1, 1, 1, 1.0), (1, 7, 5, 1.0), (3, 5, 4, 0.5), (255, 4, 16, 1.0), (256, 9, 100, 0.6),
                                                   (257, 3, 2048, 0.3), (1000, 70, 7, 0.7), (5, 300, 3, 0.5)])
def test_block_tables(pkg, rows, most, block, spare):
    rng = np.random.default_rng(rows * 131 + most)
    blocks = max(1, int(rows * most * spare))
    state = pkg.scene_pool.BlockTables(i32(np.full((rows, most), -1)), i32(np.zeros(rows)), i32(rng.permutation(blocks)), i32([blocks]), i32([0]))
    for turn in range(6):
        lengths = rng.integers(0, most * block + 1, rows)
        old = state.held.cpu().numpy()
        if turn:
            same = rng.random(rows) < 0.5
            lengths[same] = old[same]
        lengths[rng.random(rows) < 0.1] = 0
        if turn == 3:
            lengths[rng.random(rows) < 0.1] = -5
            lengths[rng.random(rows) < 0.1] = most * block + 1
        if turn == 5:
            lengths[:] = 0
        want = tables_by_rows(lengths.tolist(), block, state.tables.tolist(), old.tolist(), state.free_blocks.tolist(), int(state.n_free))
        before = [t.clone() for t in state]
        got = pkg.block_tables(i32(lengths), block, state.tables, state.held, state.free_blocks, state.n_free)
        assert all(torch.equal(a, b) for a, b in zip(before, state))      # the inputs stay
        assert got.tables.tolist() == want[0] and got.held.tolist() == want[1], turn
        assert got.free_blocks.tolist() == want[2] and got.n_free.tolist() == [want[3]] and got.status.tolist() == [want[4]], turn
        used = got.tables[got.tables >= 0].tolist() + got.free_blocks[:int(got.n_free)].tolist()
        assert sorted(used) == list(range(blocks))
        state = got
    assert int(state.n_free) == blocks


def test_block_tables_contradictory_inputs_stay_in_bounds(pkg):
    """held beyond the table, a free count beyond the stack, blocks both held and free: reported, nothing outside is touched."""
    held, n_free = i32([100, -3, 8]), i32([50])
    got = pkg.block_tables(i32([0, 4, 0]), 4, i32([[0, 1], [2, 3], [4, 5]]), held, i32([0, 1, 2, 3, 4, 5]), n_free)
    assert got.status.tolist() == [16] and got.tables.shape == (3, 2) and 0 <= int(got.n_free) <= 6


def map_by_tokens(lengths, block, tables, rows, capacity):
    slots, seq, offsets = [], [], [0]
    rows = range(len(lengths)) if rows is None else rows
    room = block * (1 if tables is None else len(tables[0]))
    for i, r in enumerate(rows):
        n = min(max(0, lengths[r]), room) if 0 <= r < len(lengths) else 0
        for p in range(n):
            page = r if tables is None else tables[r][p // block]
            slots.append(-1 if page < 0 else page * block + p % block)
            seq.append(i)
        offsets.append(offsets[-1] + n)
    fill = [-1] * max(0, capacity - len(slots))
    return offsets, (slots + fill)[:capacity], (seq + fill)[:capacity]


@pytest.mark.parametrize("scenes,points,block,picked", [(1, 1, 1, None), (1, 5000, 4096, None), (7, 900, 256, 5), (40, 300, 7, None), (3, 9000, 1000, 9),
                                                       (2000, 6, 4, 3000), (600, 3, 2, None), (5, 0, 8, 4)])
def test_slot_map(pkg, scenes, points, block, picked):
    rng = np.random.default_rng(scenes + points)
    lengths = rng.integers(0, points + 1, scenes)
    lengths[0] = points
    lengths[rng.random(scenes) < 0.2] = 0
    most = max(1, -(-points // block))
    tables = rng.permutation(scenes * most).reshape(scenes, most)
    if scenes > 3:
        tables[2, -1], lengths[3] = -1, -4
    rows = None if picked is None else rng.integers(0, scenes, picked)
    if picked is not None and picked > 2:
        rows[1], rows[2] = scenes, -1      # rows that are not there
    total = map_by_tokens(lengths.tolist(), block, tables.tolist(), None if rows is None else rows.tolist(), 0)[0][-1]
    for capacity in {total, total + 5, max(0, total - 3), total + 9000, 0}:
        for t in (tables, None):
            bs = block if t is not None else max(points, 1)
            want = map_by_tokens(lengths.tolist(), bs, None if t is None else t.tolist(), None if rows is None else rows.tolist(), capacity)
            got = pkg.slot_map(i32(lengths), bs, None if t is None else i32(t), None if rows is None else i32(rows), capacity)
            assert got.offsets.tolist() == want[0] and got.slots.tolist() == want[1] and got.sequence.tolist() == want[2], capacity
    got = pkg.slot_map(i32(lengths), block, i32(tables), None if rows is None else i32(rows))
    assert len(got.slots) == total


def test_slot_map_beyond_32_bits(pkg):
    """Slots of a pool with more than 2^31 rows: only the map is made, not the pool."""
    tables = i32([[2 ** 20 - 1, 2 ** 21], [2 ** 30, 0]])
    got = pkg.slot_map(i32([4096, 3000]), 2048, tables, capacity=7200)
    assert got.slots[0].item() == (2 ** 20 - 1) * 2048 and got.slots[2048].item() == 2 ** 21 * 2048 and got.slots[4096].item() == 2 ** 30 * 2048
    got = pkg.slot_map(i32([5] * 40000), 2 ** 30, capacity=5 * 40000)
    assert got.slots[-1].item() == 39999 * 2 ** 30 + 4


@pytest.mark.parametrize("shape,dtype", [((4,), torch.float32), ((), torch.int32), ((3,), torch.float32), ((5,), torch.float16), ((1,), torch.uint8),
                                         ((64,), torch.bfloat16), ((2, 3), torch.float64), ((257,), torch.uint8)])
def test_rows(pkg, shape, dtype):
    g = torch.Generator().manual_seed(3)
    n_src, n = 500, 777
    src = torch.randint(0, 200, (n_src,) + shape, generator=g).to(dtype).cuda()
    other = torch.randint(0, 200, (n_src, 2), generator=g).to(torch.int32).cuda()
    slots = torch.randint(-3, n_src + 3, (n,), generator=g).cuda()
    a, b = pkg.take_rows(slots, (src, other))
    there = (slots >= 0) & (slots < n_src)
    for got, s in ((a, src), (b, other)):
        want = torch.zeros((n,) + s.shape[1:], dtype=s.dtype, device="cuda")
        want[there] = s[slots[there]]
        assert torch.equal(got, want)
    assert torch.equal(pkg.take_rows(slots, (src,))[0], a)
    to = torch.randperm(900, generator=g)[:n].cuda()
    to[::7] = -1
    to[3] = 900
    dst = torch.full((900,) + shape, 7, dtype=dtype, device="cuda")
    want = dst.clone()
    go = there & (to >= 0) & (to < 900)
    want[to[go]] = src[slots[go]]
    out = pkg.put_rows(to, (src,), (dst,), source_slots=slots)
    assert out[0] is dst and torch.equal(dst, want)
    few = to[:n_src]
    go = (few >= 0) & (few < 900)
    want[few[go]] = src[go]
    pkg.put_rows(few, (src,), (dst,))
    assert torch.equal(dst, want)


def test_rows_strided_and_empty(pkg):
    wide = torch.arange(60 * 8, dtype=torch.float32, device="cuda").reshape(60, 8)
    slots = torch.tensor([5, 59, -1, 0], device="cuda")
    got, = pkg.take_rows(slots, (wide[:, 1:4],))
    assert torch.equal(got[[0, 1, 3]], wide[[5, 59, 0], 1:4]) and not got[2].any()
    got, = pkg.take_rows(slots, (wide[::2, :4],))      # 30 rows: slot 59 is outside
    assert torch.equal(got[0], wide[10, :4]) and not got[1].any()
    dst = torch.zeros((10, 8), device="cuda")
    pkg.put_rows(torch.tensor([9, 2], device="cuda"), (wide[:2, 3:5],), (dst[:, 6:],))
    assert torch.equal(dst[9, 6:], wide[0, 3:5]) and torch.equal(dst[2, 6:], wide[1, 3:5]) and not dst[:, :6].any()
    assert pkg.take_rows(slots[:0], (wide,))[0].shape == (0, 8)
    assert not pkg.take_rows(slots, (wide[:0],))[0].any()
    assert torch.equal(pkg.put_rows(slots, (wide[:0],), (dst.clone(),), source_slots=slots)[0], dst)


def test_pool_operators_on_another_stream_and_in_a_graph(pkg):
    rng = np.random.default_rng(2)
    tables, held = i32(np.full((30, 8), -1)), i32(np.zeros(30))
    free, n_free, lengths = i32(rng.permutation(200)), i32([200]), i32(rng.integers(0, 8 * 64, 30))
    src = torch.randn((30 * 512, 4), device="cuda")
    pool = torch.zeros((200 * 64, 4), device="cuda")

    def step():
        b = pkg.block_tables(lengths, 64, tables, held, free, n_free)
        m = pkg.slot_map(b.held, 64, b.tables, capacity=30 * 512)
        s = pkg.slot_map(b.held, 512, capacity=30 * 512)
        pkg.put_rows(m.slots, (src,), (pool,), source_slots=s.slots)
        return pkg.take_rows(m.slots, (pool,))[0]

    def want():
        n = lengths.tolist()
        return torch.cat([src[512 * i:512 * i + k] for i, k in enumerate(n)])

    out = step()
    assert torch.equal(out[:int(lengths.sum())], want()) and not out[int(lengths.sum()):].any()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = step()
    torch.cuda.synchronize()
    assert torch.equal(out[:int(lengths.sum())], want())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(4):
        lengths.copy_(i32(rng.integers(0, 8 * 64, 30)))
        src.normal_()
        pool.zero_()
        graph.replay()
        torch.cuda.synchronize()
        n = int(lengths.sum())
        assert torch.equal(out[:n], want()) and not out[n:].any()
        assert torch.equal(step(), out)


def _scenes(synth, n, first=0):
    """n small scenes of different lengths with two insert slots each."""
    scenes, slots, need = [], [], []
    for s in range(n):
        xyzi, label = synth.make_scene(60 + first + s, 16, 200 + 17 * s)
        scenes.append((xyzi, label))
        slots.append([[synth.make_insert(500 + 10 * (first + s), "pedestrian", rng_range=(5.0, 12.0))],
                      [synth.make_insert(501 + 10 * (first + s), "car", rng_range=(5.0, 12.0))]])
        need.append([20, 20])
    return scenes, slots, need


def _same(pool, scenes, results):
    got = pool.packed(scenes)
    offsets = got.offsets.tolist()
    for i, r in enumerate(results):
        lo, hi = offsets[i], offsets[i + 1]
        assert got.xyzi[lo:hi].cpu().numpy().tobytes() == r[0].tobytes()
        assert got.label[lo:hi].cpu().numpy().view(np.uint32).tobytes() == np.asarray(r[1]).astype(np.uint32).tobytes()
        assert (got.sequence[lo:hi] == i).all()
    assert offsets[-1] == len(got.label)


def test_pool_holds_augmented_scenes(pkg, synth):
    scenes, slots, need = _scenes(synth, 5)
    want, acc = pkg.augment_batch(scenes, slots, need)
    longest = max(len(r[0]) for r in want)
    pool = pkg.ScenePool(9, longest + 400, block_size=256)
    none, acc2 = pkg.augment_batch(scenes, slots, need, pool=pool)
    assert none is None and acc2 == acc
    _same(pool, range(5), want)
    _same(pool, [4, 0, 4, 2], [want[i] for i in (4, 0, 4, 2)])
    more, slots2, need2 = _scenes(synth, 3, 40)
    want2, _ = pkg.augment_batch(more, slots2, need2)
    pkg.augment_batch(more, slots2, need2, pool=pool, pool_scenes=[7, 0, 3])      # two of them replace others
    pool.raise_on_status()
    _same(pool, [0, 1, 2, 3, 4, 7], [want2[1], want[1], want[2], want2[2], want[4], want2[0]])
    padded = pool.packed([1, 8], capacity=len(want[1][0]) + 100)      # scene 8 is empty
    assert padded.label.shape[0] == len(want[1][0]) + 100 and not padded.xyzi[-100:].any() and (padded.slots[-100:] == -1).all()
    pool.remove([1, 3])
    assert pool.lengths.tolist()[1] == 0 and pool.lengths.tolist()[3] == 0
    _same(pool, [0, 2, 7], [want2[1], want[2], want2[0]])
    everything = sorted(pool.blocks.tables[pool.blocks.tables >= 0].tolist() + pool.blocks.free_blocks[:int(pool.blocks.n_free)].tolist())
    assert everything == list(range(len(pool.blocks.free_blocks)))
    with pytest.raises(ValueError):
        pool.packed([9])
    with pytest.raises(ValueError):
        pkg.augment_batch(more, slots2, need2, pool=pool, pool_scenes=[1, 1, 2])


def test_pool_without_room_keeps_what_it_has(pkg, synth):
    scenes, slots, need = _scenes(synth, 4)
    want, _ = pkg.augment_batch(scenes, slots, need)
    blocks = [-(-len(r[0]) // 128) for r in want]
    pool = pkg.ScenePool(4, 128 * max(blocks), n_blocks=sum(blocks[:3]), block_size=128)
    pkg.augment_batch(scenes, slots, need, pool=pool)
    with pytest.raises(pkg.R3DError):
        pool.raise_on_status()
    _same(pool, [0, 1, 2], want[:3])
    assert pool.lengths.tolist() == [len(r[0]) for r in want[:3]] + [0]


def test_from_a_batch_to_the_gradients_of_a_step(pkg, synth):
    """Scenes stay in the pool; two of them are packed, their points turned by x y z, attended within the scene, classified."""
    scenes, slots, need = _scenes(synth, 3)
    pool = pkg.ScenePool(3, 8192, block_size=512)
    want, _ = pkg.augment_batch(scenes, slots, need, pool=pool)[0], None
    assert want is None
    g = torch.Generator().manual_seed(1)
    lift, head, bias = (torch.randn(s, generator=g).cuda() * k for s, k in (((4, 64), 0.05), ((260, 64), 0.2), ((260,), 0.1)))
    batch = pool.packed([2, 0], capacity=9000)
    points = batch.xyzi[:200]      # (of the first scene: attention in full would be large)

    def step(dtype, own):
        ins = [t.to(dtype).requires_grad_() for t in (lift, head, bias)]
        x = (points.to(dtype) @ ins[0]).view(-1, 2, 32)
        if own:
            q, k = pkg.rotary_positions(x, points[:, :3], (5, 5, 5), key=x)
        else:
            freq = torch.cat([10000.0 ** (-torch.arange(5, dtype=torch.float64) / 5)] * 3).cuda()
            angle = (points[:, [0] * 5 + [1] * 5 + [2] * 5].double() * freq)[:, None]
            c, s = torch.cos(angle).to(dtype), torch.sin(angle).to(dtype)
            a, b, rest = x[..., :15], x[..., 15:30], x[..., 30:]
            q = k = torch.cat([a * c - b * s, b * c + a * s, rest], -1)
        p = torch.softmax(torch.bmm(q.transpose(0, 1).contiguous(), k.permute(1, 2, 0).contiguous()) / math.sqrt(32), -1)
        y = torch.bmm(p, x.transpose(0, 1).contiguous()).transpose(0, 1).reshape(-1, 64)
        target = batch.label[:200] & 0xFFFF
        if own:
            loss = pkg.linear_cross_entropy(y, ins[1], target, bias=ins[2], ignore_index=0)
        else:
            keep = target != 0
            logits = y @ ins[1].t() + ins[2]
            each = torch.logsumexp(logits, 1) - logits.gather(1, target.long()[:, None])[:, 0]
            loss = each[keep].sum() / keep.sum().clamp(min=1)
        return (loss.detach(), *torch.autograd.grad(loss, ins))

    own, plain = step(torch.float32, True), step(torch.float64, False)
    assert int((batch.label[:200] & 0xFFFF).max()) < 260
    for a, b in zip(own, plain):
        # a chain of seven sums of at most 260 terms in 32 bits
        assert (a.double() - b).norm() <= 7 * 260 * 2.0 ** -24 * max(b.norm().item(), 1e-3) * 8
    attended = own[1]
    assert torch.isfinite(attended).all() and attended.any()


def test_rows_beyond_32_bits(pkg):
    """A pool of 300 million points: slots, byte offsets and pages past 2^32."""
    block, most, scenes = 2048, 64, 2300
    points = block * most * scenes      # 4.8 GB of x y z i
    xyzi = torch.arange(points, dtype=torch.int32, device="cuda").view(-1, 1).expand(-1, 4).to(torch.int32).contiguous()
    tables = torch.randperm(most * scenes, generator=torch.Generator().manual_seed(1)).to(torch.int32).view(scenes, most).cuda()
    lengths = torch.full((scenes,), block * most - 7, dtype=torch.int32, device="cuda")
    m = pkg.slot_map(lengths, block, tables, capacity=points)
    n = scenes * (block * most - 7)
    assert int(m.offsets[-1]) == n and (m.slots[n:] == -1).all() and (m.sequence[n:] == -1).all()
    t = torch.arange(n, device="cuda")
    seq, p = t // (block * most - 7), t % (block * most - 7)
    assert torch.equal(m.sequence[:n], seq.int())
    assert torch.equal(m.slots[:n], tables[seq, p // block].long() * block + p % block)
    out, = pkg.take_rows(m.slots, (xyzi,))
    assert torch.equal(out[:n, 3], m.slots[:n].int()) and not out[n:].any()
    back = torch.full_like(xyzi, -5)
    pkg.put_rows(m.slots, (out,), (back,))
    named = torch.zeros(points, dtype=torch.bool, device="cuda")
    named[m.slots[:n]] = True
    assert torch.equal(back[named], xyzi[named]) and (back[~named] == -5).all()


def test_pool_calls_do_not_wait_for_the_device(pkg, synth):
    """Work that is still running when ``packed`` and ``remove`` are called is still running when they return."""
    scenes, slots, need = _scenes(synth, 3)
    pool = pkg.ScenePool(4, 8192, block_size=512)
    want, _ = pkg.augment_batch(scenes, slots, need), pkg.augment_batch(scenes, slots, need, pool=pool)
    pool.packed([1, 0], capacity=9000)      # (kernels loaded)
    pool.remove([3])
    a = torch.randn((8192, 8192), device="cuda")
    torch.cuda.synchronize()
    done = torch.cuda.Event()
    for _ in range(12):
        a = a @ a * 1e-4
    done.record()
    got = pool.packed([1, 0], capacity=9000)
    pool.remove([0])
    running = not done.query()
    torch.cuda.synchronize()
    assert running
    n = len(want[0][1][0])
    assert got.xyzi[:n].cpu().numpy().tobytes() == want[0][1][0].tobytes() and pool.lengths.tolist()[0] == 0


def test_pool_of_another_device_is_refused_before_the_work(pkg, synth):
    scenes, slots, need = _scenes(synth, 1)
    pool = pkg.ScenePool(1, 8192)
    with pytest.raises(ValueError, match="cuda:1"):
        pkg.augment_batch(scenes, slots, need, device="cuda:1", pool=pool)
    assert pool.lengths.tolist() == [0]


@pytest.mark.parametrize("scenes,points,block,empty", [(600, 10, 16, 0.0), (700, 3, 2, 0.0), (5000, 9, 4, 0.8), (900, 700, 64, 0.3), (512, 10, 16, 0.0), (513, 40, 7, 0.1)])
def test_slot_map_of_many_sequences_with_little_room(pkg, scenes, points, block, empty):
    """Capacities far below the number of tokens, and ends in the middle of what a workgroup takes."""
    rng = np.random.default_rng(scenes)
    lengths = np.full(scenes, points) if not empty else rng.integers(1, points + 1, scenes)
    lengths[rng.random(scenes) < empty] = 0
    most = -(-points // block)
    tables, rows = rng.permutation(scenes * most).reshape(scenes, most), rng.permutation(scenes)
    total = int(lengths.sum())
    offsets, slots, seq = map_by_tokens(lengths.tolist(), block, tables.tolist(), rows.tolist(), total)
    for capacity in (1, 2, 511, 2047, 2048, 2049, 2100, total // 2, total - 1):
        if capacity >= total:
            continue
        got = pkg.slot_map(i32(lengths), block, i32(tables), i32(rows), capacity)
        assert got.offsets.tolist() == offsets and got.slots.tolist() == slots[:capacity] and got.sequence.tolist() == seq[:capacity], capacity


def test_put_rows_is_seen_by_autograd(pkg):
    """A tensor that a backward pass has kept and that was written in the meantime: the pass raises, as for torch's own writes."""
    x, s = torch.randn((5, 4), device="cuda"), torch.tensor([1, 0], device="cuda")
    w = torch.ones((5, 4), device="cuda", requires_grad=True)
    y = (w * x).sum()
    before = x._version
    pkg.put_rows(s, (torch.zeros((2, 4), device="cuda"),), (x[:3],))      # (a view of it)
    assert x._version > before
    with pytest.raises(RuntimeError, match="inplace"):
        y.backward()
    y = (w * x).sum()
    pkg.put_rows(s[:0], (torch.zeros((2, 4), device="cuda"),), (x,))      # nothing is written
    y.backward()
    assert torch.equal(w.grad, x)
    with torch.inference_mode():
        z = torch.zeros((5, 4), device="cuda")
        pkg.put_rows(s, (x[:2],), (z,))
    assert torch.equal(z[:2], x[[1, 0]])


def test_pool_remembers_a_scene_without_room(pkg, synth):
    """One call that finds no room, then one that does: the status still tells, once."""
    scenes, slots, need = _scenes(synth, 2)
    pool = pkg.ScenePool(3, 8192, n_blocks=1 + 8192 // 512, block_size=512)
    pool.resize(i32([8192, 512, 1]))
    pool.resize(i32([8192, 512, 0]))
    assert pool.lengths.tolist() == [8192, 512, 0] and pool.blocks.status.tolist() == [0]
    with pytest.raises(pkg.R3DError, match="no room"):
        pool.raise_on_status()
    pool.raise_on_status()
    pool.resize(i32([0, 0, 0]))
    batch = {}
    pkg.augment_batch(scenes, slots, need, reuse=batch, pool=pool)
    pool.resize(i32([9000, 0, 0]))      # more than max_points
    pool.add(batch[2], [1, 2])
    with pytest.raises(pkg.R3DError, match="no room"):
        pool.raise_on_status()


def _equal(a, b):
    return all(p.dtype == q.dtype and p.shape == q.shape and p.tobytes() == q.tobytes() for p, q in zip(a, b)) and len(a) == len(b)


def test_scenes_without_room_come_back(pkg, synth):
    scenes, slots, need = _scenes(synth, 4)
    want, acc = pkg.augment_batch(scenes, slots, need)
    blocks = [-(-len(r[0]) // 128) for r in want]
    pool = pkg.ScenePool(6, 128 * max(blocks), n_blocks=sum(blocks[:2]), block_size=128)
    got, acc2 = pkg.augment_batch(scenes, slots, need, pool=pool, pool_scenes=[4, 1, 0, 5])
    served = pool.lengths.tolist()      # rows in order: 0, 1, 4, 5
    kept = [s for s, row in enumerate([4, 1, 0, 5]) if served[row]]
    assert acc2 == acc and 0 < len(kept) < 4
    for s in range(4):
        assert got[s] is None if s in kept else _equal(got[s], want[s])
    _same(pool, [[4, 1, 0, 5][s] for s in kept], [want[s] for s in kept])
    with pytest.raises(pkg.R3DError):
        pool.raise_on_status()


def test_pool_scenes_from_an_iterator(pkg, synth):
    scenes, slots, need = _scenes(synth, 3)
    want, _ = pkg.augment_batch(scenes, slots, need)
    pool = pkg.ScenePool(5, 8192, block_size=512)
    assert pkg.augment_batch(scenes, slots, need, pool=pool, pool_scenes=(4 - s for s in range(3)))[0] is None
    _same(pool, iter([4, 3, 2]), want)


def test_pool_takes_a_frame_of_the_level1_kernels(pkg, synth):
    """A sample of more points than the batched kernels take: its frame goes through the Level-1 kernels and from there into the pool."""
    scenes, slots, need = _scenes(synth, 3)
    slots[1][1] = [synth.make_insert(9199, "car", points=70000, centre_range=7.0, centre_az=0.7)]
    want, acc = pkg.augment_batch(scenes, slots, need)
    assert pkg.SceneBatch.last_level1 == [1]
    pool = pkg.ScenePool(4, max(len(r[0]) for r in want), block_size=512)
    none, acc2 = pkg.augment_batch(scenes, slots, need, pool=pool, pool_scenes=[3, 1, 0])
    assert none is None and [list(a) for a in acc2] == [list(a) for a in acc] and pkg.SceneBatch.last_level1 == [1]
    _same(pool, [3, 1, 0], want)
    little = pkg.ScenePool(3, pool.max_points, n_blocks=-(-len(want[0][0]) // 512), block_size=512)
    got, _ = pkg.augment_batch(scenes, slots, need, pool=little)
    assert [g is None for g in got] == [n > 0 for n in little.lengths.tolist()] and got[1] is not None
    assert all(g is None or _equal(g, w) for g, w in zip(got, want))


def test_replaced_result_refuses(pkg, synth):
    scenes, slots, need = _scenes(synth, 2)
    reuse = {}
    want, _ = pkg.augment_batch(scenes, slots, need, reuse=reuse)
    batch = reuse[2]
    batch.replace_result(0, want[1][0], want[1][1])
    again = batch.results()
    assert again[0][0].tobytes() == want[1][0].tobytes() and again[0][1].tobytes() == want[1][1].tobytes() and _equal(again[1], want[1])
    with pytest.raises(ValueError):
        batch.replace_result(0, want[1][0], want[1][1][:-1])
    with pytest.raises(ValueError):
        batch.replace_result(0, np.zeros((batch.cap + 1, 4), np.float32), np.zeros(batch.cap + 1, np.uint32))


def test_pool_used_on_another_stream_keeps_its_tables(pkg):
    """A resize on a side stream that still has work before it: the tables that it replaces are not handed out to the stream
    that the pool was made on before they have been read."""
    pool = pkg.ScenePool(2000, 64 * 16, block_size=16)
    rng = np.random.default_rng(3)
    first, second = rng.integers(0, 64 * 16 + 1, 2000), rng.integers(0, 64 * 16 + 1, 2000)
    pool.resize(i32(first))
    want = pkg.block_tables(i32(second), 16, *pool.blocks[:4])
    lengths = i32(second)
    a = torch.randn((4096, 4096), device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(10):
            a = a @ a * 1e-3
        pool.resize(lengths)
    # what the pool let go of is of these sizes: the default stream's next tensors would stand there
    other = [torch.full((n,), 77, dtype=torch.int32, device="cuda") for n in (2000 * 64, 2000 * 64, 2000, 1) for _ in range(4)]
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(pool.blocks, want)) and len(other) == 16
