"""Refusals of the pool's and the training step's operators: arguments are looked at before the GPU is (not gpu)."""
import ctypes as C

import pytest
import torch


def i32(*v):
    return torch.tensor(v, dtype=torch.int32)


def test_c_entries_refuse_without_a_gpu(pkg):
    L, lib = pkg._lib, pkg._lib.load()
    assert lib.r3d_block_tables_workspace_bytes(0) == 0 and lib.r3d_block_tables_workspace_bytes(1000) >= 4 * 2 * 8
    assert lib.r3d_block_tables(*[None] * 1, 4, 16, 2, *[None] * 3, 8, *[None] * 7, 0, None) == L.E_ARG
    assert b"block_tables" in lib.r3d_last_error()
    p = C.cast(C.create_string_buffer(64), C.c_void_p).value // 16 * 16
    bad = [(p, 0, 16, 2), (p, 4, 0, 2), (p, 4, 16, 0), (p, 4, 1 << 30, 4), (p, -1, 16, 2)]
    for lengths, rows, block, most in bad:
        assert lib.r3d_block_tables(lengths, rows, block, most, p, p, p, 8, p, p + 16, p + 16, p + 16, p + 16, None, p, 1 << 20, None) == L.E_ARG
    assert lib.r3d_block_tables(p, 4, 16, 2, p, p, p, 8, p, p, p + 16, p + 16, p + 16, None, p, 1 << 20, None) == L.E_ARG      # in place
    assert lib.r3d_block_tables(p, 4, 16, 2, p, p, p, 8, p, p + 16, p + 16, p + 16, p + 16, None, p, 8, None) == L.E_WORKSPACE
    assert lib.r3d_slot_map(None, 4, None, 16, 1, None, 4, 10, p, p, p, None) == L.E_ARG
    assert lib.r3d_slot_map(p, 4, None, 16, 1, None, 5, 10, p, p, p, None) == L.E_ARG       # five sequences of four rows
    assert lib.r3d_slot_map(p, 4, None, 16, 1, None, 4, -1, p, p, p, None) == L.E_ARG
    assert lib.r3d_slot_map(p, 4, p, 1 << 30, 4, None, 4, 10, p, p, p, None) == L.E_ARG
    assert lib.r3d_slot_map(p, 4, None, 16, 1, None, 4, 10, p, p + 8, p, None) == L.E_ARG    # alignment
    rows = (L.Rows * 1)(L.Rows(p, p, 16, 16, 16))
    assert lib.r3d_move_rows(None, 1, None, None, 1, 1, 1, None) == L.E_ARG
    assert lib.r3d_move_rows(rows, 5, None, None, 1, 1, 1, None) == L.E_ARG
    assert lib.r3d_move_rows(rows, 1, None, None, 4, 3, 4, None) == L.E_ARG
    assert lib.r3d_move_rows(rows, 1, None, None, 4, 4, 3, None) == L.E_ARG
    assert lib.r3d_move_rows((L.Rows * 1)(L.Rows(p, p, 16, 8, 16)), 1, None, None, 1, 1, 1, None) == L.E_ARG
    assert lib.r3d_rotary(None, None) == L.E_ARG
    d = L.Rotary(tokens=4, dim=8, axes=1, base=10.0, pos_type=L.T_F32)
    d.heads[0], d.sections[0] = 1, 4
    assert lib.r3d_rotary(C.byref(d), None) == L.E_ARG and b"positions" in lib.r3d_last_error()
    d.sections[0] = 5
    assert lib.r3d_rotary(C.byref(d), None) == L.E_ARG and b"pairs" in lib.r3d_last_error()
    d.sections[0], d.base = 4, -1.0
    assert lib.r3d_rotary(C.byref(d), None) == L.E_ARG
    e = L.LinearCE(n=4, v=3, d=8, ld_x=8, ld_w=8, type=L.T_F32, target_type=L.T_I64, reduction=L.CE_MEAN)
    assert all(lib.r3d_linear_ce_bytes(C.byref(e), which) > 0 for which in (0, 1, 2))
    assert lib.r3d_linear_ce_bytes(C.byref(e), 3) == 0 and lib.r3d_linear_ce_bytes(C.byref(e), -1) == 0
    assert lib.r3d_linear_ce_forward(C.byref(e), None, 0, None) == L.E_ARG
    assert lib.r3d_linear_ce_backward(C.byref(e), None, 0, None) == L.E_ARG
    for name, value in (("n", 0), ("v", 0), ("d", 0), ("ld_x", 7), ("type", L.T_F64), ("target_type", L.T_F32), ("reduction", 3), ("piece", -1)):
        old = getattr(e, name)
        setattr(e, name, value)
        assert lib.r3d_linear_ce_bytes(C.byref(e), 0) == 0, name
        setattr(e, name, old)


def test_descriptors_match_the_header(pkg):
    L = pkg._lib
    assert C.sizeof(L.Rows) == 2 * 8 + 3 * 8
    assert C.sizeof(L.Rotary) == 4 * 8 + 4 * 8 + 8 + 2 * 4 + 4 * 4 + 4 + 8 * 4 + 4 + 8 + 2 * 8 + 8
    assert C.sizeof(L.LinearCE) == 4 * 8 + 7 * 8 + 4 * 4 + 6 * 8


def test_block_tables_refuses(pkg):
    t = torch.full((4, 3), -1, dtype=torch.int32)
    good = [i32(1, 2, 3, 4), 16, t, i32(0, 0, 0, 0), i32(*range(12)), i32(12)]
    for at, value in ((0, i32(1, 2)), (0, i32(1, 2, 3, 4).long()), (1, 0), (1, 1 << 30), (2, t[:, ::2]), (2, t.reshape(-1)), (3, i32(1)),
                      (4, i32()), (5, i32(1, 2))):
        args = list(good)
        args[at] = value
        with pytest.raises(ValueError):
            pkg.block_tables(*args)
    if not torch.cuda.is_available():
        with pytest.raises(pkg.R3DError):
            pkg.block_tables(*good)


def test_slot_map_refuses(pkg):
    n, t = i32(5, 6), torch.zeros((2, 2), dtype=torch.int32)
    for args, kw in (((n.long(), 4), {}), ((n, 0), {}), ((n, 4), {"tables": t[:1]}), ((n, 4), {"tables": t.t()}), ((n, 1 << 30), {"tables": t}),
                     ((n, 4), {"rows": torch.tensor([0])}), ((n, 4), {"capacity": -1}), ((i32(), 4), {})):
        with pytest.raises(ValueError):
            pkg.slot_map(*args, **kw)
    if not torch.cuda.is_available():
        with pytest.raises(pkg.R3DError):
            pkg.slot_map(n, 4, capacity=8)


def test_rows_refuse(pkg):
    s, x = torch.zeros(3, dtype=torch.int64), torch.zeros((5, 4))
    with pytest.raises(ValueError):
        pkg.take_rows(s.int(), (x,))
    with pytest.raises(ValueError):
        pkg.take_rows(s, ())
    with pytest.raises(ValueError):
        pkg.take_rows(s, (x,) * 5)
    with pytest.raises(ValueError):
        pkg.take_rows(s, (x, x[:3]))
    with pytest.raises(ValueError):
        pkg.take_rows(s, (torch.zeros((4, 5)).t(),))
    with pytest.raises(ValueError):
        pkg.take_rows(s, (x.clone().requires_grad_(),))
    with pytest.raises(ValueError):
        pkg.put_rows(s, (x,), (x.double(),))
    with pytest.raises(ValueError):
        pkg.put_rows(s, (x[:2],), (x,))
    with pytest.raises(ValueError):
        pkg.put_rows(s, (x,), (x,), source_slots=s[:2])
    with pytest.raises(ValueError):
        pkg.put_rows(s, (x,), (x[:1].expand(5, 4),))
    if not torch.cuda.is_available():
        with pytest.raises(pkg.R3DError):
            pkg.take_rows(s, (x,))


def test_rotary_refuses(pkg):
    q, p = torch.zeros((6, 2, 16)), torch.zeros((6, 2))
    for args, kw in (((q[0], p, (4, 4)), {}), ((q, p, (4,)), {}), ((q, p[:5], (4, 4)), {}), ((q, p, (4, 5)), {}), ((q, p, (4, -1)), {}),
                     ((q, p, (4, 4)), {"style": "other"}), ((q, p, (4, 4)), {"base": 0.0}), ((q, p, (4, 4)), {"base": float("inf")}),
                     ((q, p, (4, 4)), {"key": q.half()}), ((q, p, (4, 4)), {"key": q[:5]}), ((q, p.clone().requires_grad_(), (4, 4)), {}),
                     ((torch.zeros((6, 2, 15)), p, (2, 2)), {}), ((torch.zeros((6, 1, 1024)), p, (200, 200)), {})):
        with pytest.raises(ValueError):
            pkg.rotary_positions(*args, **kw)
    for args in ((q.double(), p, (4, 4)), (q, p.to(torch.int16), (4, 4))):
        with pytest.raises(TypeError):
            pkg.rotary_positions(*args)
    if not torch.cuda.is_available():
        with pytest.raises(pkg.R3DError):
            pkg.rotary_positions(q, p, (4, 4))


def test_linear_cross_entropy_refuses(pkg):
    x, w, t = torch.zeros((6, 8)), torch.zeros((5, 8)), torch.zeros(6, dtype=torch.int64)
    for args, kw in (((x, w[:, :7], t), {}), ((x, w[:0], t), {}), ((x, w, t[:5]), {}), ((x, w, t), {"bias": torch.zeros(4)}),
                     ((x, w, t), {"reduction": "average"}), ((x, w, t), {"piece": -1}), ((x, w[0], t), {})):
        with pytest.raises(ValueError):
            pkg.linear_cross_entropy(*args, **kw)
    for args, kw in (((x, w.half(), t), {}), ((x.double(), w.double(), t), {}), ((x, w, t.float()), {}), ((x, w, t), {"bias": torch.zeros(5).half()})):
        with pytest.raises(TypeError):
            pkg.linear_cross_entropy(*args, **kw)
    if not torch.cuda.is_available():
        with pytest.raises(pkg.R3DError):
            pkg.linear_cross_entropy(x, w, t)


def test_limits_refuse_without_a_gpu(pkg):
    L, lib = pkg._lib, pkg._lib.load()
    p = C.cast(C.create_string_buffer(64), C.c_void_p).value // 16 * 16
    assert lib.r3d_block_tables_workspace_bytes(L.MAX_SCENES) > 0 and lib.r3d_block_tables_workspace_bytes(L.MAX_SCENES + 1) == 0
    assert lib.r3d_block_tables(p, L.MAX_SCENES + 1, 16, 2, p, p, p, 8, p, p + 16, p + 16, p + 16, p + 16, None, p, 1 << 40, None) == L.E_ARG
    assert lib.r3d_slot_map(p, 4, None, 16, 1, p, L.MAX_SCENES + 1, 10, p, p, p, None) == L.E_ARG
    d = L.Rotary(tokens=4, dim=8, axes=1, base=10.0, pos_type=L.T_F32, type=L.T_F32, pos=p, pos_token_stride=1, pos_axis_stride=1)
    d.sections[0], d.heads[0], d.token_stride[0], d.head_stride[0], d.x[0], d.y[0] = 4, 1, 8, 8, p + 2, p + 16
    assert lib.r3d_rotary(C.byref(d), None) == L.E_ARG and b"aligned" in lib.r3d_last_error()
    d.dim, d.heads[0], d.head_stride[0], d.token_stride[0], d.x[0] = 4096, 65536, 4096, 4096 << 16, p + 32
    d.heads[1], d.head_stride[1], d.token_stride[1], d.x[1], d.y[1] = 65536, 4096, 4096 << 16, p + 32, p + 16
    assert lib.r3d_rotary(C.byref(d), None) == L.E_ARG and b"heads" in lib.r3d_last_error()
    e = L.LinearCE(n=4, v=3, d=8, ld_x=1 << 31, ld_w=8, type=L.T_F32, target_type=L.T_I64, reduction=L.CE_MEAN)
    assert lib.r3d_linear_ce_bytes(C.byref(e), 0) == 0


def test_rows_refuse_forward_mode(pkg):
    import torch.autograd.forward_ad as fwd
    s, x = torch.zeros(3, dtype=torch.int64), torch.zeros((5, 4))
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        for call in (lambda: pkg.take_rows(s, (dual,)), lambda: pkg.put_rows(s, (dual,), (x,)), lambda: pkg.put_rows(s, (x,), (dual,))):
            with pytest.raises(ValueError, match="gradient"):
                call()


def _ce_bytes(pkg, n, v, d, kind, piece, which, **more):
    L, p = pkg._lib, 1 << 12
    e = L.LinearCE(x=p, w=p, target=p, bias=p, n=n, v=v, d=d, ld_x=d, ld_w=d, type=kind, target_type=L.T_I64, reduction=L.CE_NONE, piece=piece,
                   **{**dict(dx=p, dw=p, db=p), **more})
    size = pkg._lib.load().r3d_linear_ce_bytes(C.byref(e), which)
    assert size > 0
    return size


@pytest.mark.parametrize("n,v,d", [(9_000_000, 256, 256), (9_000_000, 288, 96), (838_000, 260, 256), (845_000, 260, 256), (2_000_000, 200, 250), (3001, 260, 128),
                                   (1_500_000, 5000, 256), (2_500_000, 5000, 160), (8192, 161280, 512), (200, 777, 160), (700, 900, 200), (20, 30000, 300),
                                   (480_000, 20, 96), (5_000_000, 20, 256), (400_000, 3000, 64), (24, 38322, 100), (100_000, 128, 640)])
def test_loss_holds_no_more_than_it_says(pkg, n, v, d):
    L, mb = pkg._lib, 2 ** 20
    up = lambda a, b: -(-a // b) * b  # noqa: E731
    rows, width, classes = up(n, 256), up(d, 64), up(v, 256)
    for kind, planes in ((L.T_F32, 3), (L.T_BF16, 1), (L.T_F16, 1)):
        for piece in (0, 1, 128, 192, 1000):
            held = rows * 2 * planes * (up(max(piece, 128), 64) if piece else 256)
            held = max(held, 512 * mb if piece == 0 else 256 * 2 * 320)      # (of a head in LDS 256 points at least)
            sums = 4 * width * (rows + classes) + 2 * 256 * mb
            if piece == 0 and planes == 1 and v <= 288 and 64 < d <= 256:      # (cut by points: no least number of classes, dx at once)
                held, sums = 512 * mb, 4 * width * classes + 256 * mb
            small = held // 32 + 16 * rows + 600 * 4 * classes + 64 * mb      # db's parts, the points' weights
            assert _ce_bytes(pkg, n, v, d, kind, piece, L.CE_BYTES_BACKWARD) <= held + sums + small, (kind, piece)
        packed = 0 if planes == 1 and d % 64 == 0 else 2 * planes * width * (n + v)
        assert _ce_bytes(pkg, n, v, d, kind, 0, L.CE_BYTES_STATE) <= 20 * n + 4 * classes + packed + 4096, kind


@pytest.mark.parametrize("n,v,d,kind", [(1_000_000, 260, 256, 1), (400_000, 288, 96, 2), (300_000, 5000, 256, 1), (100_000, 900, 200, 0)])
def test_a_smaller_piece_holds_less(pkg, n, v, d, kind):
    """(Which also says that these heads hold anything: the tests of pieces on the GPU are of the same ways.)"""
    which = pkg._lib.CE_BYTES_BACKWARD
    size = [_ce_bytes(pkg, n, v, d, kind, piece, which) for piece in (128, 256, 100000)]
    rows = n * 2 * (3 if kind == 0 else 1)      # bytes of a class
    assert size[0] < size[1] <= size[2] and size[1] - size[0] >= 100 * rows
    assert _ce_bytes(pkg, n, 260, d, 1, 0, which, dw=0, dx=0) < rows * 260


@pytest.mark.parametrize("n,v,d", [(200, 777, 160), (700, 900, 200), (300, 641, 130)])
def test_pieces_of_the_gpu_tests_are_pieces(pkg, n, v, d):
    """The heads of test_loss_pieces_of_many_classes hold less with a smaller piece: they do go piece by piece."""
    for kind in (0, 1, 2):
        size = [_ce_bytes(pkg, n, v, d, kind, piece, pkg._lib.CE_BYTES_BACKWARD, dw=0, db=0) for piece in (1, 256, 100000)]
        assert size[0] < size[1] < size[2]


@pytest.mark.skipif(torch.cuda.is_available(), reason="addresses that no GPU may be given")
def test_loss_stops_at_the_first_call_that_fails(pkg):
    """A head that takes more LDS than a kernel may without asking: without a GPU the question fails, and nothing goes on."""
    L, lib, p = pkg._lib, pkg._lib.load(), 1 << 12
    e = L.LinearCE(x=p, w=p, target=p, bias=p, n=1000, v=260, d=256, ld_x=256, ld_w=256, type=L.T_BF16, target_type=L.T_I64, reduction=L.CE_MEAN, state=p,
                   loss=p, grad=p, dx=p, dw=p, db=p)
    for call in (lib.r3d_linear_ce_forward, lib.r3d_linear_ce_backward):
        assert call(C.byref(e), p, 1 << 40, None) == L.E_HIP and b"hipFuncSetAttribute" in lib.r3d_last_error()


def test_c_entries_refuse_what_is_not_aligned(pkg):
    """(Addresses of host memory that nothing is launched for.)"""
    L, lib = pkg._lib, pkg._lib.load()
    p = C.cast(C.create_string_buffer(256), C.c_void_p).value // 64 * 64 + 64
    assert lib.r3d_block_tables(p, 4, 16, 2, p, p, p, 8, p, p + 16, p + 16, p + 16, p + 16, None, p + 4, 1 << 20, None) == L.E_ARG
    assert lib.r3d_slot_map(p, 4, None, 16, 1, None, 4, 10, p + 4, p, p, None) == L.E_ARG
    rows = (L.Rows * 1)(L.Rows(p, p, 16, 16, 16))
    assert lib.r3d_move_rows(rows, 1, p + 4, None, 1, 1, 1, None) == L.E_ARG and lib.r3d_move_rows(rows, 1, None, p + 4, 1, 1, 1, None) == L.E_ARG
    d = L.Rotary(tokens=4, dim=8, axes=1, base=10.0, pos_type=L.T_F64, type=L.T_F32, pos=p + 4, pos_token_stride=1, pos_axis_stride=1)
    d.sections[0], d.heads[0], d.token_stride[0], d.head_stride[0], d.x[0], d.y[0] = 4, 1, 8, 8, p, p + 16
    assert lib.r3d_rotary(C.byref(d), None) == L.E_ARG and b"aligned" in lib.r3d_last_error()
    good = dict(x=p, w=p, target=p, bias=p, state=p, loss=p, grad=p, dx=p, dw=p, db=p, workspace=p)
    for name, by in (("x", 1), ("w", 1), ("bias", 1), ("dx", 1), ("dw", 1), ("db", 1), ("target", 4), ("loss", 2), ("grad", 2), ("state", 8), ("workspace", 8)):
        at = dict(good, **{name: p + by})
        ws = at.pop("workspace")
        e = L.LinearCE(n=4, v=3, d=8, ld_x=8, ld_w=8, type=L.T_BF16, target_type=L.T_I64, reduction=L.CE_MEAN, **at)
        for call in (lib.r3d_linear_ce_forward, lib.r3d_linear_ce_backward):
            assert call(C.byref(e), ws, 1 << 40, None) == L.E_ARG and b"aligned" in lib.r3d_last_error(), name


def test_rotary_in_c_refuses_a_base_that_is_not_finite(pkg):
    L, lib = pkg._lib, pkg._lib.load()
    p = C.cast(C.create_string_buffer(256), C.c_void_p).value // 64 * 64 + 64
    d = L.Rotary(tokens=4, dim=8, axes=1, pos_type=L.T_F32, type=L.T_F32, pos=p, pos_token_stride=1, pos_axis_stride=1)
    d.sections[0], d.heads[0], d.token_stride[0], d.head_stride[0], d.x[0], d.y[0] = 4, 1, 8, 8, p, p + 16
    for base in (float("inf"), float("nan"), 0.0, -2.0):
        d.base = base
        assert lib.r3d_rotary(C.byref(d), None) == L.E_ARG and b"base" in lib.r3d_last_error()


def test_pool_knows_its_device_by_number(pkg, monkeypatch):
    """"cuda" is the device that is current when the pool is made, for the pool and for the batch that is to go into it."""
    pool = object.__new__(pkg.ScenePool)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    pool.device = pkg.scene_pool._with_index("cuda")
    assert pool.device == torch.device("cuda:1")
    pool.check_device("cuda")
    pool.check_device("cuda:1")
    for other in ("cuda:0", "cpu"):
        with pytest.raises(ValueError, match="the pool on cuda:1"):
            pool.check_device(other)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    with pytest.raises(ValueError):
        pool.check_device("cuda")


def test_rows_refuse_a_tensor_for_a_tuple(pkg):
    s, x = torch.zeros(3, dtype=torch.int64), torch.zeros((4, 4))
    for call in (lambda: pkg.take_rows(s, x), lambda: pkg.put_rows(s, x, (x,)), lambda: pkg.put_rows(s, (x,), x)):
        with pytest.raises(ValueError, match="tuple"):
            call()
