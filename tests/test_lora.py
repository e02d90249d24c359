"""Low-rank adapters of many requests beside a shared projection (`oxs_lora_add`).

The GPU results are compared with y + B (s A x) in 64 bits. u = 2^-24 is half a
step of a float relative to its value; products are exact, so
- v_r = s sum_k A x is off by at most (k / 16 + 32) u sum |A| |x| |s|: no term
  passes more than k / 16 + 30 additions (a wavefront's 64 lanes, or the 16
  products of a matrix instruction, are summed as trees), and the scale rounds once;
- the delta adds |B| times that, and (R + 8) u sum |B| |v| for its own sum;
- y is rounded once: u |y| for float32, 2^-8 |y| for bfloat16 (half a step), with u |y| for the sum.
"""
import ctypes

import numpy as np
import pytest

from oxide_sampler import _abi

U = 2.0 ** -24


def reference(y, x, ids, adapters, bf16_out=False):
    """(result, bound) in float64; adapters: {slot: (a, b, scale)} with [rank, k] and [m, rank] tensors."""
    out = y.double().clone()
    bound = out.abs() * 0
    for slot, (a, b, scale) in adapters.items():
        rows = (ids == slot).nonzero()[:, 0]
        if len(rows) == 0:
            continue
        a, b, xs, s = a.double(), b.double(), x[rows].double(), float(np.float32(scale))
        rank, k = a.shape
        v = (xs @ a.T) * s
        v_off = (xs.abs() @ a.abs().T) * abs(s) * ((k / 16 + 32) * U)
        out[rows] += v @ b.T
        bound[rows] = (v_off + v.abs() * ((rank + 8) * U)) @ b.abs().T
        bound[rows] += out[rows].abs() * (U + (2.0 ** -8 if bf16_out else 0)) + 1e-40
    return out, bound


def make(torch, seed, batch, m, k, ranks, dtype="bf16", scale=None):
    """x, y and an adapter for every slot (rank 0: none)."""
    t = torch
    dt = {"f32": t.float32, "bf16": t.bfloat16, "f16": t.float16}[dtype]
    g = t.Generator(device="cuda").manual_seed(seed)
    x = t.randn(batch, k, generator=g, device="cuda") * 1.5
    y = t.randn(batch, m, generator=g, device="cuda") * 3
    ad = {}
    for i, r in enumerate(ranks):
        if r:
            ad[i] = ((t.randn(r, k, generator=g, device="cuda") / k ** 0.5).to(dt),
                     t.randn(m, r, generator=g, device="cuda").to(dt), 0.25 * (i % 5 + 1) if scale is None else scale)
    return x, y, ad, dt, g


def table(t, m, k, ranks, ad, dt, batch, max_rank=None):
    from oxide_sampler import LoraAdapters
    lora = LoraAdapters(m, k, max_adapters=len(ranks), max_rank=max_rank or max(max(ranks), 1), max_batch=batch,
                        dtype=dt)
    for i, (a, b, s) in ad.items():
        lora.load(i, a, b, s)
    return lora


def check(got, want, bound, what=""):
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), f"{what}: off {float((off - bound).max())} beyond the bound"


# ------------------------------------------------------------------ on the CPU: what the calls refuse

@pytest.fixture()
def lib():
    return _abi.load_library()


def valid():
    t = _abi.OxsLoraTable(100, 64, 4, 16, _abi.OXS_DTYPE_BF16, 4096, 8192, 12288, 16384)
    b = _abi.OxsLoraBatch(2, _abi.OXS_DTYPE_F32, _abi.OXS_DTYPE_F32, 4096, 64, 8192, 100, 12288, 16384, 1 << 20)
    return t, b


TABLE_FAULTS = [{"m": 0}, {"k": 0}, {"max_adapters": 0}, {"max_adapters": 65537}, {"max_rank": 0}, {"max_rank": 257},
                {"m": (1 << 30) + 1}, {"k": (1 << 30) + 1}, {"dtype": 3}, {"dtype": -1}]


@pytest.mark.parametrize("change", TABLE_FAULTS)
def test_refused_tables(lib, change):
    t, b = valid()
    for f, v in change.items():
        setattr(t, f, v)
    n = ctypes.c_size_t()
    assert lib.oxs_lora_table_bytes(t, n, n) == _abi.OXS_ERR_INVALID_ARGUMENT
    assert lib.oxs_lora_workspace_bytes(t, 1) == 0
    assert lib.oxs_lora_add(t, b, None) == _abi.OXS_ERR_INVALID_ARGUMENT
    assert lib.oxs_lora_load(t, 0, 4096, 64, 4096, 16, 16, 1.0, None) == _abi.OXS_ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("change", [{"a": None}, {"b": None}, {"ranks": None}, {"scales": None}, {"a": 4104},
                                    {"b": 8200}, {"ranks": 2}, {"scales": 1}])
def test_refused_table_pointers(lib, change):
    t, b = valid()
    for f, v in change.items():
        setattr(t, f, v)
    assert lib.oxs_lora_add(t, b, None) == _abi.OXS_ERR_INVALID_ARGUMENT
    assert lib.oxs_lora_load(t, 0, 4096, 64, 4096, 16, 16, 1.0, None) == _abi.OXS_ERR_INVALID_ARGUMENT
    n = ctypes.c_size_t()
    assert lib.oxs_lora_table_bytes(t, n, n) == _abi.OXS_OK  # its pointers are not looked at


@pytest.mark.parametrize("change,code", [
    ({"x": None}, _abi.OXS_ERR_INVALID_ARGUMENT), ({"y": None}, _abi.OXS_ERR_INVALID_ARGUMENT),
    ({"adapters": None}, _abi.OXS_ERR_INVALID_ARGUMENT), ({"workspace": None}, _abi.OXS_ERR_INVALID_ARGUMENT),
    ({"x_ld": 63}, _abi.OXS_ERR_INVALID_ARGUMENT), ({"y_ld": 99}, _abi.OXS_ERR_INVALID_ARGUMENT),
    ({"y_ld": -100}, _abi.OXS_ERR_INVALID_ARGUMENT), ({"x_dtype": 2}, _abi.OXS_ERR_INVALID_ARGUMENT),
    ({"y_dtype": 2}, _abi.OXS_ERR_INVALID_ARGUMENT), ({"y_dtype": 7}, _abi.OXS_ERR_INVALID_ARGUMENT),
    ({"x": 4098}, _abi.OXS_ERR_INVALID_ARGUMENT), ({"y": 4097, "y_dtype": 1}, _abi.OXS_ERR_INVALID_ARGUMENT),
    ({"adapters": 4098}, _abi.OXS_ERR_INVALID_ARGUMENT), ({"workspace": 4100}, _abi.OXS_ERR_INVALID_ARGUMENT),
    ({"workspace_bytes": 16}, _abi.OXS_ERR_INVALID_ARGUMENT), ({"batch": 65537}, _abi.OXS_ERR_LIMITS),
])
def test_refused_batches(lib, change, code):
    t, b = valid()
    for f, v in change.items():
        setattr(b, f, v)
    assert lib.oxs_lora_add(t, b, None) == code


def test_refused_loads_and_empty_calls(lib):
    t, b = valid()
    bad = _abi.OXS_ERR_INVALID_ARGUMENT
    ok = dict(slot=0, a=4096, a_ld=64, b=8192, b_ld=16, rank=16)
    for change in ({"slot": 4}, {"rank": 17}, {"a": None}, {"b": None}, {"a": 4097}, {"b": 8193}, {"a_ld": 63},
                   {"b_ld": 15}):
        c = {**ok, **change}
        assert lib.oxs_lora_load(t, c["slot"], c["a"], c["a_ld"], c["b"], c["b_ld"], c["rank"], 1.0, None) == bad, change
    assert lib.oxs_lora_add(t, None, None) == bad and lib.oxs_lora_add(None, b, None) == bad
    assert lib.oxs_lora_load(None, 0, 4096, 64, 8192, 16, 16, 1.0, None) == bad
    assert lib.oxs_lora_table_bytes(t, None, None) == bad
    b.batch = 0
    assert lib.oxs_lora_add(t, b, None) == _abi.OXS_OK
    big = _abi.OxsLoraTable(1 << 30, 64, 4, 16, _abi.OXS_DTYPE_BF16, 4096, 8192, 12288, 16384)
    b.batch, b.y_ld, b.workspace_bytes = 65536, 1 << 30, 1 << 40
    assert lib.oxs_lora_add(big, b, None) == _abi.OXS_ERR_LIMITS


def test_table_and_workspace_sizes(lib):
    # large tables are counted in 64 bits, and more of anything never needs less
    a, b = ctypes.c_size_t(), ctypes.c_size_t()
    t = _abi.OxsLoraTable(262144, 8192, 4096, 256, _abi.OXS_DTYPE_F32)
    assert lib.oxs_lora_table_bytes(t, a, b) == _abi.OXS_OK
    assert a.value >= 8192 * 4096 * 256 * 4 and b.value >= 262144 * 4096 * 256 * 4
    sizes = [lib.oxs_lora_workspace_bytes(t, n) for n in (1, 2, 31, 32, 33, 64, 1000, 65536)]
    assert sizes[0] > 0 and sizes == sorted(sizes)
    assert lib.oxs_lora_workspace_bytes(t, 65537) == 0


# ------------------------------------------------------------------ on the GPU

CASES = [
    # batch, m, k, ranks of the slots, weights, x, y
    (1, 1, 1, [1], "f32", "f32", "f32"),
    (1, 5, 3, [2], "bf16", "bf16", "bf16"),
    (2, 31, 31, [1, 3], "f16", "f32", "f32"),
    (3, 33, 64, [8, 0, 7], "bf16", "f32", "f32"),
    (1, 1000, 896, [16], "bf16", "f32", "f32"),
    (1, 1001, 895, [15], "f32", "bf16", "bf16"),
    (5, 127, 129, [16, 17], "bf16", "bf16", "f32"),
    (7, 129, 1000, [9, 33, 16, 1], "f16", "f32", "bf16"),
    (24, 4099, 895, [8] * 24, "f32", "f32", "f32"),
    (31, 2048, 512, [16, 32, 8], "bf16", "f32", "f32"),
    (32, 640, 256, [64], "f16", "bf16", "bf16"),
    (33, 514, 130, [4] * 40, "bf16", "f32", "bf16"),
    (64, 3000, 2048, [16, 8] * 8, "bf16", "f32", "f32"),
    (65, 257, 4096, [64, 16, 5], "bf16", "bf16", "f32"),
    (100, 1024, 96, [128, 100], "f32", "f32", "f32"),
    (130, 511, 72, [256, 3], "bf16", "f32", "f32"),
    (40, 1500, 4096, [48, 0, 16], "f16", "f32", "f32"),
    (300, 700, 200, [16] * 9, "f16", "f32", "f32"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["mixed", "packed"])
@pytest.mark.parametrize("batch,m,k,ranks,w,xd,yd", CASES)
def test_matches_the_definition(torch_gpu, batch, m, k, ranks, w, xd, yd, order):
    t = torch_gpu
    x, y, ad, dt, g = make(t, batch * 13 + m, batch, m, k, ranks, w)
    kinds = {"f32": t.float32, "bf16": t.bfloat16}
    x, y = x.to(kinds[xd]), y.to(kinds[yd])
    # slots, slots past the table, and none; one adapter alone when there is one row
    ids = t.randint(0, len(ranks) + 1, (batch,), generator=g, device="cuda", dtype=t.int32)
    ids[t.rand(batch, generator=g, device="cuda") < 0.1] = -1
    if batch == 1:
        ids[:] = 0
    if order == "packed":
        ids = ids.sort().values
    want, bound = reference(y, x, ids, ad, yd == "bf16")
    before = y.clone()
    lora = table(t, m, k, ranks, ad, dt, batch)
    assert lora.add(y, x, ids) is y
    check(y, want, bound, f"{batch} x {m}")
    idle = t.tensor([int(i) not in ad for i in ids.tolist()], device="cuda")
    assert t.equal(y[idle], before[idle])


@pytest.mark.gpu
@pytest.mark.parametrize("batch,ranks,w", [(47, [16] * 5, "bf16"), (48, [8, 3], "f32"), (49, [16] * 5, "bf16"),
                                           (1023, [4] * 3, "f16"), (1024, [16], "bf16"), (1025, [5, 16], "f32"),
                                           (2100, [8, 0, 20], "bf16"), (3000, [2] * 100, "bf16")])
@pytest.mark.parametrize("order", ["mixed", "packed", "falling"])
def test_batches_around_the_kernels_own_sizes(torch_gpu, batch, ranks, w, order):
    t = torch_gpu
    m, k = 200, 40
    x, y, ad, dt, g = make(t, batch, batch, m, k, ranks, w)
    ids = t.randint(-1, len(ranks) + 1, (batch,), generator=g, device="cuda", dtype=t.int32)
    if order != "mixed":
        ids = ids.sort(descending=order == "falling").values
    want, bound = reference(y, x, ids, ad)
    table(t, m, k, ranks, ad, dt, batch).add(y, x, ids)
    check(y, want, bound, f"{batch} {order}")


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["mixed", "packed"])
@pytest.mark.parametrize("batch,m,k,ranks,w,xd,yd", CASES)
def test_small_tables_slots_for_large_ranks(torch_gpu, batch, m, k, ranks, w, xd, yd, order):
    # with room for rank 256 and more inputs the same calls take two launches and tiles of 8 rows
    t = torch_gpu
    k += 640
    x, y, ad, dt, g = make(t, batch * 17 + m, batch, m, k, ranks, w)
    kinds = {"f32": t.float32, "bf16": t.bfloat16}
    x = x.to(kinds[xd])
    flat = t.full((batch, m + batch % 5), 7.0, dtype=kinds[yd], device="cuda")  # y of many alignments
    yv = flat[:, :m]
    yv.copy_(y)
    ids = t.randint(-1, len(ranks) + 1, (batch,), generator=g, device="cuda", dtype=t.int32)
    if batch == 1:
        ids[:] = 0
    if order == "packed":
        ids = ids.sort().values
    want, bound = reference(yv, x, ids, ad, yd == "bf16")
    before = flat.clone()
    lora = table(t, m, k, ranks, ad, dt, batch, max_rank=256)
    lora.add(yv, x, ids)
    check(yv, want, bound, f"{batch} x {m}")
    idle = t.tensor([int(i) not in ad for i in ids.tolist()], device="cuda")
    assert t.equal(flat[idle], before[idle]) and t.equal(flat[:, m:], before[:, m:])


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [3, 40])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_infinities_stay_with_their_rows_in_small_tiles(torch_gpu, batch, dtype):
    t = torch_gpu
    m, k, ranks = 700, 1000, [16, 16, 3]
    x, y, ad, dt, g = make(t, 78, batch, m, k, ranks, dtype)
    ids = t.randint(0, 3, (batch,), generator=g, device="cuda", dtype=t.int32)
    ids[:3] = t.tensor([0, 1, 2])
    want, bound = reference(y, x, ids, ad)
    bad = ad | {1: (ad[1][0].clone(), ad[1][1].clone(), ad[1][2])}
    bad[1][0][3, 5] = float("inf")
    bad[1][1][2, 4] = float("nan")
    x[0, 999] = float("nan")  # the last value of an odd eight
    table(t, m, k, ranks, bad, dt, batch, max_rank=256).add(y, x, ids)
    fine = ids != 1
    fine[0] = False
    check(y[fine], want[fine], bound[fine])
    assert bool(y[0].isnan().all()) and not bool(y[ids == 1].isfinite().any())


LARGE = [
    # tiles of 32 rows: batch, m, k, ranks of the slots, weights, x, y, extra elements between y's rows
    (33, 70001, 24, [16, 3], "f32", "f32", "f32", 0),
    (65, 40000, 40, [16] * 40, "bf16", "bf16", "f32", 1),
    (96, 50257, 512, [8, 17], "bf16", "f32", "bf16", 0),
    (97, 40002, 30, [5, 0, 64], "f32", "f32", "bf16", 2),
    (150, 36003, 64, [33, 16, 2], "f16", "f32", "f32", 5),
    (257, 16500, 9, [16] * 20, "f16", "bf16", "bf16", 3),
    (300, 12001, 77, [256, 1], "bf16", "f32", "f32", 3),
    (1024, 4100, 20, [12, 16], "bf16", "f32", "f32", 4),
    (1025, 4099, 16, [4] * 9, "f32", "bf16", "f32", 1),
    (2100, 2500, 33, [8, 0, 20], "bf16", "f32", "bf16", 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["mixed", "packed"])
@pytest.mark.parametrize("batch,m,k,ranks,w,xd,yd,pad", LARGE)
def test_large_tiles_match_the_definition(torch_gpu, batch, m, k, ranks, w, xd, yd, pad, order):
    t = torch_gpu
    kinds = {"f32": t.float32, "bf16": t.bfloat16}
    x, y, ad, dt, g = make(t, batch * 3 + m, batch, m, k, ranks, w)
    x = x.to(kinds[xd])
    flat = t.full((batch, m + pad), 7.0, dtype=kinds[yd], device="cuda")
    yv = flat[:, :m]
    yv.copy_(y)
    ids = t.randint(-1, len(ranks) + 1, (batch,), generator=g, device="cuda", dtype=t.int32)
    if order == "packed":
        ids = ids.sort().values
    want, bound = reference(yv, x, ids, ad, yd == "bf16")
    before = flat.clone()
    table(t, m, k, ranks, ad, dt, batch).add(yv, x, ids)
    check(yv, want, bound, f"{batch} x {m}")
    idle = t.tensor([int(i) not in ad for i in ids.tolist()], device="cuda")
    assert t.equal(flat[idle], before[idle]) and t.equal(flat[:, m:], before[:, m:])


@pytest.mark.gpu
@pytest.mark.parametrize("m,k", [(50257, 895), (129, 4095), (6, 513)])
@pytest.mark.parametrize("w", ["f32", "bf16", "f16"])
def test_one_row_of_odd_sizes(torch_gpu, m, k, w):
    t = torch_gpu
    x, y, ad, dt, g = make(t, m, 1, m, k, [0, 31], w)
    ids = t.ones(1, dtype=t.int32, device="cuda")
    lora = table(t, m, k, [0, 31], ad, dt, 1)
    for shift in (0, 1, 4):
        yv = t.full((m + 8,), 7.0, device="cuda")
        xv = t.full((k + 8,), float("nan"), device="cuda")
        yv[shift:shift + m], xv[shift:shift + k] = y[0], x[0]
        want, bound = reference(y, x, ids, ad)
        lora.add(yv[shift:shift + m][None], xv[shift:shift + k][None], ids)
        check(yv[shift:shift + m][None], want, bound, f"shift {shift}")
        assert bool((yv[:shift] == 7).all()) and bool((yv[shift + m:] == 7).all())


@pytest.mark.gpu
@pytest.mark.parametrize("xd,yd,xpad,ypad,xshift,yshift", [("f32", "f32", 1, 3, 1, 1), ("bf16", "bf16", 5, 1, 3, 1),
                                                           ("f32", "f32", 4, 4, 0, 0), ("bf16", "f32", 8, 2, 8, 2),
                                                           ("f32", "bf16", 2, 8, 2, 4)])
def test_strides_and_alignment_leave_the_gaps_alone(torch_gpu, xd, yd, xpad, ypad, xshift, yshift):
    t = torch_gpu
    kinds = {"f32": t.float32, "bf16": t.bfloat16}
    for batch, m, k in ((40, 1000, 300), (3, 130, 77), (70, 256, 64)):
        x, y, ad, dt, g = make(t, batch, batch, m, k, [16, 5, 24], "bf16")
        xs = t.full((xshift + batch * (k + xpad),), float("nan"), dtype=kinds[xd], device="cuda")
        ys = t.full((yshift + batch * (m + ypad),), 7.0, dtype=kinds[yd], device="cuda")
        xv = xs[xshift:].view(batch, k + xpad)[:, :k]
        yv = ys[yshift:].view(batch, m + ypad)[:, :m]
        xv.copy_(x)
        yv.copy_(y)
        ids = t.randint(0, 3, (batch,), generator=g, device="cuda", dtype=t.int32)
        want, bound = reference(yv, xv, ids, ad, yd == "bf16")
        table(t, m, k, [16, 5, 24], ad, dt, batch).add(yv, xv, ids)
        check(yv, want, bound)
        assert bool((ys[:yshift] == 7).all()) and bool((ys[yshift:].view(batch, m + ypad)[:, m:] == 7).all())


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [6, 40, 200])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_infinities_and_nan_stay_with_their_rows(torch_gpu, batch, dtype):
    t = torch_gpu
    m, k, ranks = 700, 320, [16, 16, 3]
    x, y, ad, dt, g = make(t, 77, batch, m, k, ranks, dtype)
    ids = t.randint(0, 3, (batch,), generator=g, device="cuda", dtype=t.int32)
    ids[:6] = t.tensor([0, 1, 2, 1, -1, 0])
    want, bound = reference(y, x, ids, ad)
    bad = ad | {1: (ad[1][0].clone(), ad[1][1].clone(), ad[1][2])}
    bad[1][0][3, 5] = float("inf")
    bad[1][1][2, 4] = float("nan")
    x[5, 7] = float("nan")
    x[0, 1] = float("inf")
    table(t, m, k, ranks, bad, dt, batch).add(y, x, ids)
    fine = t.ones(batch, dtype=t.bool, device="cuda")
    fine[ids == 1] = False
    fine[5] = fine[0] = False
    check(y[fine], want[fine], bound[fine])
    assert bool(y[5].isnan().all()) and not bool(y[0].isfinite().any())
    assert not bool(y[ids == 1].isfinite().any())  # an infinite value of v meets weights of every output


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,yd", [("f32", "f32"), ("bf16", "f32"), ("f16", "bf16")])
def test_a_bad_adapter_beside_others_in_large_tiles(torch_gpu, dtype, yd):
    # enough rows and outputs for tiles of 32 rows, each of several adapters; y of odd and of even strides
    t = torch_gpu
    batch, k, ranks = 200, 72, [16, 20, 3, 0, 9]
    for m in (20001, 26000):
        x, y, ad, dt, g = make(t, m, batch, m, k, ranks, dtype)
        y = y.to(t.float32 if yd == "f32" else t.bfloat16)
        ids = t.randint(-1, 5, (batch,), generator=g, device="cuda", dtype=t.int32)
        want, bound = reference(y, x, ids, ad, yd == "bf16")
        bad = ad | {1: (ad[1][0], ad[1][1].clone(), ad[1][2])}
        bad[1][1][::3, 17] = float("inf")
        bad[1][1][1::3, 0] = float("nan")
        before = y.clone()
        table(t, m, k, ranks, bad, dt, batch).add(y, x, ids)
        fine = ids != 1
        check(y[fine], want[fine], bound[fine], f"m={m}")
        assert not bool(y[~fine][:, ::3].isfinite().any()) and bool(y[~fine][:, 1::3].isnan().all())
        check(y[~fine][:, 2::3], want[~fine][:, 2::3], bound[~fine][:, 2::3], f"m={m}, outputs of finite weights")
        assert t.equal(y[(ids < 0) | (ids == 3)], before[(ids < 0) | (ids == 3)])


@pytest.mark.gpu
def test_wide_ranges_of_values(torch_gpu):
    # large and tiny weights and values beside each other: no term is lost to a narrower format
    t = torch_gpu
    for dtype, lo, hi in (("f32", 1e-12, 1e12), ("bf16", 1e-12, 1e12), ("f16", 1e-4, 1e3)):
        x, y, ad, dt, g = make(t, 5, 33, 600, 256, [16, 8], dtype)
        x *= t.logspace(-6, 6, 256, device="cuda")
        a, b, s = ad[0]
        ad[0] = ((a.float() * t.logspace(6, -6, 256, device="cuda").clamp(lo, hi)).to(dt),
                 (b.float() * t.logspace(-3, 2, 16, device="cuda")).to(dt), s)
        ids = t.arange(33, dtype=t.int32, device="cuda") % 2
        want, bound = reference(y, x, ids, ad)
        table(t, 600, 256, [16, 8], ad, dt, 33).add(y, x, ids)
        check(y, want, bound, dtype)


@pytest.mark.gpu
def test_small_terms_are_not_rounded_away(torch_gpu):
    # one value of x with 24 significant bits through weights of 1: y is exact
    t = torch_gpu
    from oxide_sampler import LoraAdapters
    for dt in (t.float32, t.bfloat16, t.float16):
        for batch in (1, 33):
            lora = LoraAdapters(300, 64, 1, 16, batch, dt)
            a, b = t.zeros(1, 64, dtype=dt, device="cuda"), t.ones(300, 1, dtype=dt, device="cuda")
            a[0, 9] = 1
            lora.load(0, a, b)
            x = t.zeros(batch, 64, device="cuda")
            x[:, 9] = t.arange(batch, device="cuda") + (2.0 ** 23 + 1) / 2 ** 23 + 2.0 ** 10
            x[:, 9] = x[:, 9].nextafter(t.tensor(9e9, device="cuda"))
            y = t.zeros(batch, 300, device="cuda")
            lora.add(y, x, t.zeros(batch, dtype=t.int32, device="cuda"))
            assert t.equal(y, x[:, 9:10].expand(batch, 300)), dt


@pytest.mark.gpu
def test_slots_change_in_stream_order_and_under_a_graph(torch_gpu):
    t = torch_gpu
    m, k, batch, ranks = 900, 256, 40, [8, 16, 0]
    x, y, ad, dt, g = make(t, 9, batch, m, k, ranks)
    lora = table(t, m, k, ranks, ad, dt, batch, max_rank=40)
    other = table(t, m, k, ranks, ad, dt, batch, max_rank=40)  # a table and workspace of its own
    ids = t.randint(0, 3, (batch,), generator=g, device="cuda", dtype=t.int32)
    y0 = y.clone()
    call = lora.descriptor(y, x, ids)
    yo = y.clone()
    other_call = other.descriptor(yo, x, ids)
    graphs = []
    for obj, c in ((lora, call), (other, other_call)):
        gr = t.cuda.CUDAGraph()
        with t.cuda.graph(gr):
            obj.launch(c)
        graphs.append(gr)
    side = t.cuda.Stream()
    new = make(t, 10, batch, m, k, [40, 3, 12])[2]
    for i in range(4):
        if i == 1:  # another adapter in slot 0, of another rank
            lora.load(0, *new[0])
            ad[0] = new[0]
        if i == 2:
            lora.unload(1)
            del ad[1]
            lora.load(2, *new[2])
            ad[2] = new[2]
        y.copy_(y0)
        yo.copy_(y0)
        want, bound = reference(y0, x, ids, ad)
        side.wait_stream(t.cuda.current_stream())
        graphs[0].replay()
        with t.cuda.stream(side):
            graphs[1].replay()
        t.cuda.synchronize()
        check(y, want, bound, f"replay {i}")
        eager = lora.add(y0.clone(), x, ids)
        assert t.equal(y, eager)
        if i == 0:
            assert t.equal(yo, y)


@pytest.mark.gpu
@pytest.mark.parametrize("batch,m", [(1, 700), (5, 700), (9, 3000), (100, 30000), (1025, 5000)])
def test_rows_behind_the_last_stay_as_they_were(torch_gpu, batch, m):
    t = torch_gpu
    x, y, ad, dt, g = make(t, m, batch + 40, m, 48, [16, 7])
    ids = t.randint(0, 2, (batch + 40,), generator=g, device="cuda", dtype=t.int32)
    want, bound = reference(y[:batch], x[:batch], ids[:batch], ad)
    behind = y[batch:].clone()
    lora = table(t, m, 48, [16, 7], ad, dt, batch + 40)
    lora.add(y[:batch], x[:batch], ids[:batch])
    check(y[:batch], want, bound)
    assert t.equal(y[batch:], behind)


@pytest.mark.gpu
def test_two_calls_on_one_table_at_once(torch_gpu):
    # the table is read only: a workspace each is all that two streams need
    t = torch_gpu
    m, k, batch, ranks = 20000, 512, 100, [16, 8, 30]
    x, y, ad, dt, g = make(t, 31, batch, m, k, ranks)
    lora = table(t, m, k, ranks, ad, dt, batch)
    ids = t.randint(0, 3, (batch,), generator=g, device="cuda", dtype=t.int32)
    want = lora.add(y.clone(), x, ids)
    second = t.empty_like(lora.workspace)
    streams = [t.cuda.Stream(), t.cuda.Stream()]
    ys = [[y.clone() for _ in range(6)] for _ in streams]
    calls = [[lora.descriptor(z, x, ids) for z in zs] for zs in ys]
    for c in calls[1]:
        c.workspace = second.data_ptr()
    for s in streams:
        s.wait_stream(t.cuda.current_stream())
    for i in range(6):
        for s, cs in zip(streams, calls):
            lora.launch(cs[i], s)
    t.cuda.synchronize()
    for zs in ys:
        for z in zs:
            assert t.equal(z, want)


@pytest.mark.gpu
def test_another_stream_and_repeated_calls(torch_gpu):
    t = torch_gpu
    x, y, ad, dt, g = make(t, 3, 50, 1200, 300, [16, 16])
    lora = table(t, 1200, 300, [16, 16], ad, dt, 50)
    ids = t.randint(0, 2, (50,), generator=g, device="cuda", dtype=t.int32)
    want = lora.add(y.clone(), x, ids)
    for _ in range(3):
        assert t.equal(lora.add(y.clone(), x, ids), want)
    s = t.cuda.Stream()
    z = y.clone()
    s.wait_stream(t.cuda.current_stream())
    lora.add(z, x, ids, stream=s)
    s.synchronize()
    assert t.equal(z, want)
    # fewer rows than the object was made for
    assert t.equal(lora.add(y[:7].clone(), x[:7], ids[:7]), want[:7])


@pytest.mark.gpu
def test_offsets_past_32_bits(torch_gpu):
    t = torch_gpu
    m, k, ld = 500, 64, (1 << 30) + 12
    x, y, ad, dt, g = make(t, 21, 5, m, k, [16, 4])
    flat = t.empty(4 * ld + m, dtype=t.bfloat16, device="cuda")
    yv = flat.as_strided((5, m), (ld, 1))
    yv.copy_(y)
    ids = t.tensor([0, 1, -1, 1, 0], dtype=t.int32, device="cuda")
    want, bound = reference(yv, x, ids, ad, True)
    table(t, m, k, [16, 4], ad, dt, 5).add(yv, x, ids)
    check(yv, want, bound)


@pytest.mark.gpu
def test_a_table_past_32_bits(torch_gpu):
    # the last of the slots lies past 4 GiB in both halves of the table
    t = torch_gpu
    from oxide_sampler import LoraAdapters
    m, k, n = 40000, 40960, 900
    lora = LoraAdapters(m, k, n, 64, 4, t.bfloat16)
    x, y, ad, dt, g = make(t, 2, 4, m, k, [64, 40])
    lora.load(0, *ad[0])
    lora.load(n - 1, *ad[1])
    ids = t.tensor([n - 1, 0, n - 2, n - 1], dtype=t.int32, device="cuda")
    want, bound = reference(y, x, ids, {0: ad[0], n - 1: ad[1]})
    lora.add(y, x, ids)
    check(y, want, bound)


@pytest.mark.gpu
def test_python_refusals(torch_gpu):
    t = torch_gpu
    from oxide_sampler import LoraAdapters
    with pytest.raises(TypeError):
        LoraAdapters(10, 10, 1, 4, 1, t.float64)
    for sizes in ((0, 10, 1, 4, 1), (10, 10, 0, 4, 1), (10, 10, 1, 4, 0), (10, 10, 1, 4, 70000)):
        with pytest.raises(ValueError):
            LoraAdapters(*sizes)
    with pytest.raises(_abi.OxsError):
        LoraAdapters(10, 10, 1, 257, 1)
    lora = LoraAdapters(40, 32, 2, 8, 3)
    a = t.zeros(8, 32, dtype=t.bfloat16, device="cuda")
    b = t.zeros(40, 8, dtype=t.bfloat16, device="cuda")
    x, y = t.zeros(3, 32, device="cuda"), t.zeros(3, 40, device="cuda")
    ids = t.zeros(3, dtype=t.int32, device="cuda")
    for call in (lambda: lora.load(0, a.float(), b), lambda: lora.load(0, a, b.t()), lambda: lora.load(0, a[:4], b),
                 lambda: lora.load(0, a[:, :31], b), lambda: lora.load(0, a.cpu(), b),
                 lambda: lora.load(0, a[:1].expand(8, 32), b),
                 lambda: lora.add(y.half(), x, ids), lambda: lora.add(y, x[:, :31], ids),
                 lambda: lora.add(y, x, ids.long()), lambda: lora.add(y, x, ids[:2]), lambda: lora.add(y.cpu(), x, ids),
                 lambda: lora.add(y[:1].expand(3, 40), x, ids), lambda: lora.add(y.t(), x, ids),
                 lambda: lora.add(t.zeros(4, 40, device="cuda"), t.zeros(4, 32, device="cuda"), ids)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: lora.load(2, a, b), lambda: lora.unload(-1)):
        with pytest.raises(IndexError):
            call()
    y += 1
    assert bool((lora.add(y, x, ids) == 1).all())  # no slot is loaded
    assert lora.add(y[:0], x[:0], ids[:0]).shape == (0, 40)


@pytest.mark.gpu
def test_the_whole_step_together(torch_gpu):
    """Quantize -> shared Q8_0 projection with adapters -> decode step -> log probabilities, as a server runs them;
    captured and replayed too. Rows without an adapter keep the projection's exact logits."""
    from oxide_sampler import DecodeLoop, LmHeadQ8_0, quantize_q8_1
    from test_lm_head import random_case
    from test_logprobs import check as check_logprobs, reference as logprobs_reference
    t = torch_gpu
    m, k, S = 2000, 256, 12
    rng = np.random.default_rng(6)
    w, x = random_case(rng, m, k, S)
    head = LmHeadQ8_0(w, m, k)
    xs = t.from_numpy(x).cuda()
    _, _, ad, dt, g = make(t, 4, S, m, k, [16, 8, 4], scale=0.5)
    lora = table(t, m, k, [16, 8, 4], ad, dt, S)
    ids = t.tensor([0, 1, 2, -1, 0, 1, 2, -1, 0, 0, 1, -1], dtype=t.int32, device="cuda")
    xq = quantize_q8_1(xs)
    base = head.project(xq)
    logits = t.empty(S, m, device="cuda")

    loop = DecodeLoop(S, m, top_logprobs=5)
    for s in range(S):
        loop.add_sequence(s, temperature=0.0 if s % 3 == 0 else 0.8, top_p=0.9, current_token=1, current_position=0,
                          max_tokens=100)

    def step():
        quantize_q8_1(xs, out=xq)
        head.project(xq, out=logits, adapters=lora, x=xs, row_adapters=ids)

    want, bound = reference(base, xs, ids, ad)
    graph = t.cuda.CUDAGraph()
    for i in range(4):
        if i == 2:
            with t.cuda.graph(graph):
                step()
            loop.capture(logits)
        logits.zero_()
        if i < 2:
            step()
            loop.step(logits)
        else:
            graph.replay()
            loop.step()
        t.cuda.synchronize()
        check(logits, want, bound)
        assert t.equal(logits[ids < 0], base[ids < 0])
        tokens = loop.out["tokens"].cpu().numpy()
        host = logits.cpu().numpy()
        check_logprobs({n: v.cpu().numpy() for n, v in loop.logprobs.items()},
                       logprobs_reference(host, tokens[:, None], 5), m)
        greedy = np.arange(S) % 3 == 0
        np.testing.assert_array_equal(tokens[greedy], host[greedy].argmax(axis=1))
    loop.close()
    for bad in (dict(adapters=lora), dict(x=xs), dict(adapters=lora, x=xs)):
        with pytest.raises(ValueError):
            head.project(xq, **bad)
    with pytest.raises(ValueError):
        head.project(xq, adapters=table(t, m, 128, [1], {}, dt, S), x=xs, row_adapters=ids)
