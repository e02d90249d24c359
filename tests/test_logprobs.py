"""Token log probabilities, ranks, entropy and alternatives (`oxs_token_logprobs`).

The GPU results are compared with the definition in 64 bits (numpy). Ranks,
alternatives' ids and statuses have to be equal; the floats lie within
`tolerances`, derived from the operations' roundings:
u = 2^-24 is half a step of a float relative to its value. A difference to the
row's largest logit, its scaling and the change of the exponential's base round
q relatively by at most 5u, which moves e^q relatively by 5u |q|; the hardware's
exponential adds 2u, a sum of n terms in any order at most n u. A thread sums
at most V / 256 + 64 terms one after the other.
"""
import ctypes

import numpy as np
import pytest

from oxide_sampler import _abi, workloads as wl

U = 2.0 ** -24
NINF = -np.inf


def present_logits(x, mask):
    """float64 logits with -inf for the tokens that are not present."""
    x = x.astype(np.float64)
    x[np.isnan(x)] = NINF
    if mask is not None:
        x[~mask] = NINF
    return x


def reference(x, tokens, top, mask=None, temperatures=None, softcap=0.0):
    """The definition in 64 bits, of float32 (or widened bf16) logits [rows, V]."""
    l = present_logits(x, mask)
    rows, V = l.shape
    y = l.copy()
    if softcap > 0:
        y = np.where(l == NINF, NINF, softcap * np.tanh(l / softcap))
    if temperatures is not None:
        t = np.where(temperatures > 1e-6, temperatures, 1.0).astype(np.float64)
        y = np.where(y == NINF, NINF, y / t[:, None])
    out = {k: np.zeros(rows) for k in ("logsumexp", "entropy", "mean_q")}
    out["status"] = np.zeros(rows, np.int32)
    T = 0 if tokens is None else tokens.shape[1]
    out["logprobs"], out["ranks"] = np.zeros((rows, T)), np.zeros((rows, T), np.int32)
    out["top_ids"], out["top_logprobs"] = np.full((rows, top), -1, np.int32), np.full((rows, top), NINF)
    for b in range(rows):
        m = y[b].max()
        if m == NINF:
            lse, ent = NINF, 0.0
            lp = np.full(V, NINF)
            out["status"][b] = 1
        elif m == np.inf:
            lse, ent = np.inf, np.nan
            lp = np.where(y[b] == np.inf, np.nan, NINF)
        else:
            q = y[b] - m
            e = np.exp(q)
            s = e.sum()
            qe = np.where(e > 0, np.where(np.isfinite(q), q, 0.0) * e, 0.0).sum()
            lse, ent = m + np.log(s), np.log(s) - qe / s
            lp = q - np.log(s)
            out["mean_q"][b] = -qe / s
        out["logsumexp"][b], out["entropy"][b] = lse, ent
        here = np.flatnonzero(l[b] > NINF)
        order = here[np.argsort(-l[b][here], kind="stable")]  # equal logits stay in order of their ids
        n = min(top, len(order))
        out["top_ids"][b, :n], out["top_logprobs"][b, :n] = order[:n], lp[order[:n]]
        for j in range(T):
            t = int(np.uint32(tokens[b, j]))
            if t >= V or l[b, t] == NINF:
                out["logprobs"][b, j] = NINF
                continue
            out["logprobs"][b, j] = lp[t]
            out["ranks"][b, j] = 1 + (l[b] > l[b, t]).sum() + (l[b, :t] == l[b, t]).sum()
    return out


def tolerances(ref, V, softcap=0.0, temperatures=None):
    """Absolute bounds per row for logsumexp, entropy and, beside 6u per unit of their value, log probabilities."""
    n = V / 256 + 64
    cap = 0.0
    if softcap > 0:  # division, tanh (4 half steps) and product round y by 6u cap at most
        inv = 1.0 if temperatures is None else 1.0 / np.where(temperatures > 1e-6, temperatures, 1.0)
        cap = 2 * 6 * U * softcap * inv
    ln_s = (n + 5 * ref["mean_q"] + 4) * U + cap
    fin = np.where(np.isfinite(ref["logsumexp"]), np.abs(ref["logsumexp"]), 0.0)
    return {"logsumexp": ln_s + 4 * U * fin, "entropy": (2 * ln_s + 8 * U) * (1 + np.nan_to_num(ref["entropy"])),
            "logprobs": ln_s + cap}


def bf16(x):
    return wl.bf16_bits_to_f32(wl.f32_to_bf16_bits(x))


def check(got, ref, V, softcap=0.0, temperatures=None, what=""):
    tol = tolerances(ref, V, softcap, temperatures)
    for name in ("status", "ranks", "top_ids"):
        if name in got:
            np.testing.assert_array_equal(got[name].reshape(ref[name].shape), ref[name], err_msg=f"{what} {name}")
    for name in ("logsumexp", "entropy", "logprobs", "top_logprobs"):
        if name not in got:
            continue
        g, r = got[name].reshape(ref[name].shape).astype(np.float64), ref[name].copy()
        r[np.abs(r) > np.finfo(np.float32).max] *= np.inf  # what a float rounds it to
        sure = np.isfinite(r)
        np.testing.assert_array_equal(g[~sure], r[~sure], err_msg=f"{what} {name}")
        t = tol["logprobs" if name == "top_logprobs" else name]
        t = np.broadcast_to(t[:, None] if r.ndim == 2 else t, r.shape)
        if name in ("logprobs", "top_logprobs"):
            t = t + 6 * U * np.abs(np.where(sure, r, 0.0))
        off = np.abs(g[sure] - r[sure])
        assert (off <= t[sure]).all(), f"{what} {name}: off {off.max()} (bound {t[sure][off.argmax()]})"


def run(torch, x, tokens=None, top=0, mask=None, temperatures=None, softcap=0.0, dtype="f32", pad=0, shift=0,
        lp=None, **kw):
    """One call over host arrays; pad: extra elements between rows; shift: elements before the first row."""
    from oxide_sampler import TokenLogprobs
    rows, V = x.shape
    dt = torch.float32 if dtype == "f32" else torch.bfloat16
    flat = torch.full((shift + rows * (V + pad),), float("nan"), dtype=dt, device="cuda")
    logits = flat[shift:].view(rows, V + pad)[:, :V]
    logits.copy_(torch.from_numpy(x).to(dt))
    dev = lambda a: None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    words = None if mask is None else dev(wl.pack_mask(mask, V).view(np.int32))
    if mask is not None and mask.shape[0] == 1 and rows > 1:
        words = words[0]
    lp = lp or TokenLogprobs()
    out = lp.compute(logits, dev(None if tokens is None else tokens.astype(np.int64).astype(np.uint32).view(np.int32)),
                     top=top, mask=words, temperatures=dev(temperatures), softcap=softcap, **kw)
    torch.cuda.synchronize()
    return {k: v.cpu().numpy() for k, v in out.items()}


def special_rows(V, rng):
    """Rows where a softmax goes wrong: name -> float32 logits [V]."""
    n = rng.standard_normal(V).astype(np.float32) * 3
    low = np.finfo(np.float32).min
    r = {"normal": n, "all -inf": np.full(V, NINF), "all nan": np.full(V, np.nan), "equal": np.full(V, 1.5),
         "zeros of both signs": np.where(np.arange(V) % 3 == 0, -0.0, 0.0), "all lowest": np.full(V, low),
         "one": np.full(V, NINF), "ascending": np.arange(V) * 0.001, "descending": -np.arange(V) * 0.001,
         "infinities and nan": n.copy(), "plus inf": n.copy(), "all plus inf": np.full(V, np.inf),
         "lowest but three": np.full(V, low), "far apart": n.copy(), "large": n * 1e4, "tiny": n * 1e-6,
         "few values": np.round(n)}
    r["one"][V // 2] = -7.0
    r["infinities and nan"][rng.random(V) < 0.5] = NINF
    r["infinities and nan"][rng.random(V) < 0.3] = np.nan
    r["plus inf"][[V // 3, V - 1]] = np.inf
    r["lowest but three"][[0, V // 2, V - 1]] = [1.0, 2.0, 1.0]
    r["far apart"][V // 4] = 3e38
    r["far apart"][V // 5] = -3e38
    return {k: np.asarray(v, np.float32) for k, v in r.items()}


def some_tokens(x, T, rng):
    """Per row: the likeliest, the last, random ones and one outside the vocabulary."""
    rows, V = x.shape
    t = rng.integers(0, V, (rows, T)).astype(np.int64)
    if T > 1:
        t[:, 0] = np.nan_to_num(x, nan=NINF).argmax(axis=1)
        t[:, 1] = V - 1
    if T > 3:
        t[:, 2] = V
        t[:, 3] = t[:, 0]  # a token given twice
    return t


# ------------------------------------------------------------------ on the CPU: what the call refuses

@pytest.fixture()
def lib():
    return _abi.load_library()


def valid_call():
    """A descriptor that passes every check (its addresses are never used by a refused call)."""
    d = _abi.OxsLogprobs()
    d.rows, d.vocab, d.logits_dtype, d.tokens_per_row, d.top_n = 2, 100, _abi.OXS_DTYPE_F32, 1, 4
    d.logits_ld, d.tokens_ld, d.mask_ld = 100, 1, 4
    for i, f in enumerate(("logits", "tokens", "allowed_mask", "temperatures", "out_logprobs", "out_ranks",
                           "out_logsumexp", "out_entropy", "out_top_ids", "out_top_logprobs", "out_status",
                           "workspace")):
        setattr(d, f, 4096 * (i + 1))
    d.workspace_bytes = _abi.load_library().oxs_logprobs_workspace_bytes()
    return d


@pytest.mark.parametrize("change,code", [
    ({"vocab": 0}, _abi.OXS_ERR_SHAPE_MISMATCH),
    ({"vocab": (1 << 30) + 1, "logits_ld": 1 << 31, "mask_ld": 0}, _abi.OXS_ERR_LIMITS),
    ({"rows": (1 << 23) + 1}, _abi.OXS_ERR_LIMITS),
    ({"tokens_per_row": 65, "tokens_ld": 65}, _abi.OXS_ERR_LIMITS),
    ({"top_n": 33}, _abi.OXS_ERR_LIMITS),
    ({"logits_dtype": 2}, _abi.OXS_ERR_INVALID_ARGUMENT),
    ({"logits_dtype": -1}, _abi.OXS_ERR_INVALID_ARGUMENT),
    ({"logits": None}, _abi.OXS_ERR_INVALID_ARGUMENT),
    ({"tokens": None}, _abi.OXS_ERR_INVALID_ARGUMENT),
    ({"workspace": None}, _abi.OXS_ERR_INVALID_ARGUMENT),
    ({"logits_ld": 99}, _abi.OXS_ERR_INVALID_ARGUMENT),
    ({"logits_ld": -100}, _abi.OXS_ERR_INVALID_ARGUMENT),
    ({"tokens_ld": 0}, _abi.OXS_ERR_INVALID_ARGUMENT),
    ({"mask_ld": 3}, _abi.OXS_ERR_INVALID_ARGUMENT),
    ({"mask_ld": -1}, _abi.OXS_ERR_INVALID_ARGUMENT),
    ({"logits": 4098}, _abi.OXS_ERR_INVALID_ARGUMENT),
    ({"logits_dtype": _abi.OXS_DTYPE_BF16, "logits": 4097}, _abi.OXS_ERR_INVALID_ARGUMENT),
    ({"tokens": 4097}, _abi.OXS_ERR_INVALID_ARGUMENT),
    ({"out_top_ids": 4098}, _abi.OXS_ERR_INVALID_ARGUMENT),
    ({"workspace": 4104}, _abi.OXS_ERR_INVALID_ARGUMENT),
    ({"workspace_bytes": 15}, _abi.OXS_ERR_INVALID_ARGUMENT),
])
def test_refused_calls(lib, change, code):
    d = valid_call()
    for f, v in change.items():
        setattr(d, f, v)
    assert lib.oxs_token_logprobs(d, None) == code


def test_refuses_no_call_and_ignores_no_rows(lib):
    assert lib.oxs_token_logprobs(None, None) == _abi.OXS_ERR_INVALID_ARGUMENT
    d = valid_call()
    d.rows = 0
    assert lib.oxs_token_logprobs(d, None) == _abi.OXS_OK


def test_struct_matches_the_header(tmp_path):
    from test_abi import HEADER
    import re
    import subprocess
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    structs = {"oxs_logprobs": _abi.OxsLogprobs, "oxs_lora_table": _abi.OxsLoraTable,
               "oxs_lora_batch": _abi.OxsLoraBatch}
    lines = ["#include <stddef.h>", "#include <stdio.h>", f'#include "{HEADER}"', "int main(void) {"]
    for name, cls in structs.items():
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, flags=re.S).group(1)
        assert re.findall(r"(\w+)\s*;", body) == [f for f, _ in cls._fields_], name
        lines.append(f'  printf("%zu\\n", sizeof({name}));')
        lines += [f'  printf("%zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["  return 0;", "}"]) + "\n")
    subprocess.run(["gcc", "-std=c11", "-o", str(exe), str(src)], check=True)
    want = []
    for cls in structs.values():
        want += [ctypes.sizeof(cls)] + [getattr(cls, f).offset for f, _ in cls._fields_]
    got = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()
    assert [int(v) for v in got] == want
    src_py = (HEADER.parent.parent / "oxide-tech-llm-engine_amd" / "oxide_sampler" / "_abi.py").read_text()
    for name in ("OXS_LOGPROBS_MAX_TOP", "OXS_LOGPROBS_MAX_TOKENS", "OXS_LORA_MAX_RANK", "OXS_LORA_NONE",
                 "OXS_DTYPE_F16"):
        assert int(re.search(r"#define %s (\w+?)u?\b" % name, text).group(1), 0) == getattr(_abi, name), name
        assert name in src_py


def test_reference_closed_forms():
    # two equal logits: each ln(1/2), entropy ln 2, the lower id first
    r = reference(np.array([[3.0, 3.0, NINF]], np.float32), np.array([[1, 2]]), 3)
    np.testing.assert_allclose(r["logprobs"][0, 0], -np.log(2), rtol=1e-15)
    assert r["logprobs"][0, 1] == NINF and r["ranks"].tolist() == [[2, 0]] and r["top_ids"].tolist() == [[0, 1, -1]]
    np.testing.assert_allclose([r["entropy"][0], r["logsumexp"][0]], [np.log(2), 3 + np.log(2)], rtol=1e-15)
    # n equal logits at any temperature: entropy ln n; a cap's image is one value too
    r = reference(np.full((1, 50), 8.0, np.float32), None, 0, temperatures=np.array([0.3], np.float32), softcap=5.0)
    np.testing.assert_allclose(r["entropy"][0], np.log(50), rtol=1e-14)


# ------------------------------------------------------------------ on the GPU

CASES = [
    # rows, V, dtype, T, top, mask, temperatures, softcap, pad, shift
    (1, 1, "f32", 1, 1, None, False, 0.0, 0, 0),
    (3, 2, "bf16", 2, 5, None, True, 0.0, 0, 0),
    (2, 31, "f32", 4, 32, 0.5, False, 0.0, 1, 0),
    (5, 33, "f32", 5, 7, 0.5, True, 4.0, 3, 1),
    (1, 257, "bf16", 1, 20, None, False, 0.0, 0, 3),
    (4, 1000, "f32", 0, 20, None, False, 0.0, 0, 0),
    (4, 1023, "bf16", 64, 0, 0.9, False, 30.0, 9, 0),
    (1, 4097, "f32", 16, 32, None, True, 0.0, 0, 1),
    (2, 8191, "bf16", 3, 31, 0.01, False, 0.0, 1, 1),
    (7, 8192, "f32", 1, 1, None, False, 0.0, 0, 0),
    (3, 8193, "f32", 2, 17, None, False, 0.0, 3, 0),
    (1, 32000, "f32", 1, 5, None, False, 0.0, 0, 0),
    (1, 32000, "bf16", 1, 32, 0.03, True, 15.0, 8, 0),
    (24, 50257, "f32", 4, 0, None, False, 30.0, 6, 0),
    (9, 65537, "bf16", 2, 20, 0.3, False, 0.0, 7, 0),
    (64, 40000, "f32", 1, 20, None, False, 0.0, 0, 0),
    (70, 16385, "bf16", 1, 8, 0.03, True, 0.0, 0, 0),
    (300, 5003, "f32", 1, 3, None, True, 0.0, 0, 2),
    (600, 3001, "bf16", 2, 2, None, False, 0.0, 5, 0),
    (1200, 2050, "f32", 1, 0, 0.5, False, 0.0, 0, 0),
    (2100, 1030, "bf16", 1, 4, None, False, 0.0, 2, 0),
    (2, 262147, "f32", 2, 20, None, False, 0.0, 0, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,V,dtype,T,top,mask,temps,softcap,pad,shift", CASES)
def test_matches_the_definition(torch_gpu, rows, V, dtype, T, top, mask, temps, softcap, pad, shift):
    rng = np.random.default_rng(rows * 7 + V)
    x = wl.zipf_prior_logits(rng, min(rows, 40), V, 3.0)
    x = np.ascontiguousarray(x[np.arange(rows) % len(x)])
    x += rng.standard_normal((rows, 1)).astype(np.float32)
    if dtype == "bf16":
        x = bf16(x)
    m = None
    if mask is not None:
        m = rng.random((rows, V)) < mask
        m[rows // 2] = False  # a row whose mask leaves nothing
        if rows > 3:
            m[1] = False
            m[1, [0, V - 1]] = True  # and one with fewer tokens than alternatives
    t = rng.uniform(0.3, 2.0, rows).astype(np.float32) if temps else None
    if temps:
        t[0] = 0.0  # a greedy row
    tokens = some_tokens(x, T, rng) if T else None
    got = run(torch_gpu, x, tokens, top, m, t, softcap, dtype, pad, shift)
    check(got, reference(x, tokens, top, m, t, softcap), V, softcap, t, f"rows={rows} V={V}")


@pytest.mark.gpu
@pytest.mark.parametrize("rows,V,dtype,T,top", [(3, 40000, "f32", 64, 5), (1, 262147, "bf16", 64, 32),
                                                (200, 70001, "bf16", 9, 0), (141, 90000, "f32", 17, 7),
                                                (511, 300001, "bf16", 3, 1), (16, 128256, "f32", 8, 10),
                                                (11, 128256, "f32", 2, 11), (149, 8100, "f32", 33, 3)])
def test_split_rows_with_many_tokens(torch_gpu, rows, V, dtype, T, top):
    rng = np.random.default_rng(V + T)
    x = bf16(wl.zipf_prior_logits(rng, min(rows, 8), V, 3.0))[np.arange(rows) % min(rows, 8)]
    x[rows // 2, ::2] = NINF
    t = rng.uniform(0.5, 2.0, rows).astype(np.float32)
    tokens = some_tokens(x, T, rng)
    n = min(rows, 8)  # (the rows repeat: the reference of the first and of the changed one is enough)
    pick = np.unique(np.r_[np.arange(n), rows // 2, rows - 1])
    got = run(torch_gpu, x, tokens, top, temperatures=t, dtype=dtype)
    ref = reference(x[pick], tokens[pick], top, temperatures=t[pick])
    check({k: v[pick] for k, v in got.items()}, ref, V, temperatures=t[pick], what=f"rows={rows} V={V}")


@pytest.mark.gpu
@pytest.mark.parametrize("V,dtype", [(5, "f32"), (100, "bf16"), (1500, "f32"), (9000, "bf16"), (33000, "f32")])
@pytest.mark.parametrize("top", [0, 3, 32])
def test_special_rows(torch_gpu, V, dtype, top):
    rng = np.random.default_rng(V + top)
    named = special_rows(V, rng)
    x = np.stack(list(named.values()))
    if dtype == "bf16":
        finite = np.isfinite(x)
        x = np.where(finite, bf16(np.where(finite, x, 0).clip(-3.38e38, 3.38e38)), x).astype(np.float32)
    tokens = some_tokens(x, 5, rng)
    with np.errstate(all="ignore"):
        ref = reference(x, tokens, top)
        got = run(torch_gpu, x, tokens, top, dtype=dtype)
    for b, name in enumerate(named):
        one = lambda r: {k: v[b:b + 1] for k, v in r.items()}  # noqa: E731
        check(one(got), one(ref), V, what=name)


@pytest.mark.gpu
def test_many_rows_of_special_values(torch_gpu):
    # as many rows as make each row one workgroup's
    V, rng = 4100, np.random.default_rng(5)
    base = np.stack(list(special_rows(V, rng).values()))
    x = base[np.arange(2048) % len(base)]
    tokens = some_tokens(x, 2, rng)
    with np.errstate(all="ignore"):
        ref = reference(x[:len(base)], tokens[:len(base)], 6)
        got = run(torch_gpu, x, tokens, 6)
        check({k: v[:len(base)] for k, v in got.items()}, ref, V, what="first rows")
    for k in ("top_ids", "top_logprobs", "entropy", "logsumexp", "status"):
        np.testing.assert_array_equal(got[k], got[k][np.arange(2048) % len(base)], err_msg=k)


@pytest.mark.gpu
def test_one_mask_for_all_rows(torch_gpu):
    rng = np.random.default_rng(11)
    x = rng.standard_normal((6, 5000)).astype(np.float32)
    m = rng.random((1, 5000)) < 0.2
    tokens = some_tokens(x, 3, rng)
    got = run(torch_gpu, x, tokens, 9, m)
    check(got, reference(x, tokens, 9, np.repeat(m, 6, axis=0)), 5000)


@pytest.mark.gpu
def test_mask_bits_past_the_vocabulary_are_ignored(torch_gpu):
    from oxide_sampler import TokenLogprobs
    t = torch_gpu
    x = t.randn(3, 37, device="cuda")
    buf = t.full((3, 40), 50.0, device="cuda")
    buf[:, :37] = x
    full = t.full((3, 2), -1, dtype=t.int32, device="cuda")
    lp = TokenLogprobs()
    ref = reference(x.cpu().numpy(), None, 32)
    for out in (lp.compute(buf[:, :37], top=32, mask=full), lp.compute(x, top=32)):
        check({k: v.cpu().numpy() for k, v in out.items()}, ref, 37)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,V", [(16, 1), (16, 30), (9, 33), (9, 2047), (9, 8200), (40, 32769), (600, 20001)])
def test_masks_of_rows_on_every_boundary(torch_gpu, rows, V, dtype):
    # odd strides: the rows begin on every element boundary of 16 bytes, and their masks' words on none of them
    rng = np.random.default_rng(V)
    x = bf16(rng.standard_normal((min(rows, 40), V)).astype(np.float32))[np.arange(rows) % min(rows, 40)]
    m = rng.random((rows, V)) < rng.random((rows, 1))
    m[0], m[-1] = True, False
    m[1], m[2] = np.arange(V) == V - 1, np.arange(V) == 0
    tokens = some_tokens(x, 3, rng)
    for pad in (1 if V % 2 == 0 else 0, 8 - V % 8):
        got = run(torch_gpu, x, tokens, 4, m, dtype=dtype, pad=pad)
        check(got, reference(x, tokens, 4, m), V, what=f"pad {pad}")
        got = run(torch_gpu, x, tokens, 0, m, dtype=dtype, pad=pad)
        check(got, reference(x, tokens, 0, m), V, what=f"pad {pad}, no alternatives")


@pytest.mark.gpu
@pytest.mark.parametrize("temp", [1e-7, 1e-6, 2e-6, 1e-3, 50.0, float("inf"), float("nan"), -1.0])
def test_temperatures_at_the_edges(torch_gpu, temp):
    rng = np.random.default_rng(3)
    x = rng.standard_normal((2, 3000)).astype(np.float32)
    t = np.full(2, temp, np.float32)
    with np.errstate(all="ignore"):
        ref = reference(x, some_tokens(x, 2, np.random.default_rng(1)), 4, temperatures=t)
    check(run(torch_gpu, x, some_tokens(x, 2, np.random.default_rng(1)), 4, temperatures=t), ref, 3000)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,V", [(4, 1500), (3, 33000), (600, 900)])
def test_softcaps_at_the_edges(torch_gpu, rows, V, dtype):
    rng = np.random.default_rng(V)
    x = bf16(wl.zipf_prior_logits(rng, rows, V, 3.0))
    x[:, ::7] = 0.0
    x[0, 3:] = NINF
    tokens = some_tokens(x, 4, rng)
    got = run(torch_gpu, x, tokens, 5, softcap=1e-40, dtype=dtype)  # every logit becomes 0 to 40 places
    check(got, reference(x, tokens, 5, softcap=1e-40), V)
    plain = run(torch_gpu, x, tokens, 5, dtype=dtype)
    got = run(torch_gpu, x, tokens, 5, softcap=np.inf, dtype=dtype)  # tends to no cap
    for name in plain:
        np.testing.assert_array_equal(got[name], plain[name], err_msg=name)
    # 1e30 is as good as none: the division, the series and the product round y by 4u |l| at most, and of a log
    # probability's or the entropy's terms three hold a y
    got, ref = run(torch_gpu, x, tokens, 5, softcap=1e30, dtype=dtype), reference(x, tokens, 5)
    most = 12 * U * np.abs(x[np.isfinite(x)]).max()
    tol = tolerances(ref, V)
    for name, bound in (("logsumexp", tol["logsumexp"]), ("logprobs", tol["logprobs"][:, None])):
        r = ref[name]
        fin = np.isfinite(r)
        np.testing.assert_array_equal(got[name][~fin], r[~fin].astype(np.float32))
        off = np.abs(got[name][fin] - r[fin])
        assert (off <= np.broadcast_to(bound, r.shape)[fin] + most + 6 * U * np.abs(r[fin])).all(), name


@pytest.mark.gpu
def test_only_the_asked_outputs_are_written(torch_gpu):
    from oxide_sampler import TokenLogprobs
    t = torch_gpu
    x = t.randn(5, 3000, device="cuda")
    tok = t.arange(15, dtype=t.int32, device="cuda").view(5, 3)
    lp = TokenLogprobs()
    whole = lp.compute(x, tok, top=4)
    guard = {k: t.full((v.numel() + 64,), 77, dtype=v.dtype, device="cuda") for k, v in whole.items()}
    out = {k: guard[k][32:32 + v.numel()].view(v.shape) for k, v in whole.items()}
    lp.compute(x, tok, top=4, out=out)
    for k, v in whole.items():
        assert t.equal(out[k], v), k
        assert bool((guard[k][:32] == 77).all()) and bool((guard[k][32 + v.numel():] == 77).all()), k
    # a raw call that leaves every output out but one
    for keep in whole:
        d, o = lp.descriptor(x, tok, top=4)
        for k in whole:
            if k != keep:
                setattr(d, "out_" + k, None)
        o[keep].fill_(0)
        lp.launch(d)
        assert t.equal(o[keep], whole[keep]), keep


@pytest.mark.gpu
def test_offsets_past_32_bits(torch_gpu):
    from oxide_sampler import TokenLogprobs
    t = torch_gpu
    rows, V, ld = 5, 4001, (1 << 30) + 8
    flat = t.empty((rows - 1) * ld + V, dtype=t.bfloat16, device="cuda")
    logits = flat.as_strided((rows, V), (ld, 1))
    x = bf16(np.random.default_rng(2).standard_normal((rows, V)).astype(np.float32) * 3)
    logits.copy_(t.from_numpy(x))
    tokens = some_tokens(x, 2, np.random.default_rng(9))
    out = TokenLogprobs().compute(logits, t.from_numpy(tokens.astype(np.int32)).cuda(), top=6)
    check({k: v.cpu().numpy() for k, v in out.items()}, reference(x, tokens, 6), V)


@pytest.mark.gpu
def test_graphs_streams_and_repeats(torch_gpu):
    from oxide_sampler import TokenLogprobs
    t = torch_gpu
    g = t.Generator(device="cuda").manual_seed(4)
    sets = [(t.randn(r, v, generator=g, device="cuda") * 3, t.randint(0, v, (r, 1), generator=g, device="cuda",
                                                                      dtype=t.int32)) for r, v in
            ((2, 70001), (40, 9000))]
    eager = [TokenLogprobs().compute(x, k, top=7) for x, k in sets]
    graphs = []
    for x, k in sets:
        lp = TokenLogprobs()
        call, out = lp.descriptor(x, k, top=7)
        gr = t.cuda.CUDAGraph()
        with t.cuda.graph(gr):
            lp.launch(call)
        graphs.append((gr, out, lp))
    side = t.cuda.Stream()
    side.wait_stream(t.cuda.current_stream())
    for i in range(4):  # one graph on each stream at once, eager work between
        with t.cuda.stream(side):
            graphs[0][0].replay()
        graphs[1][0].replay()
        sets[0][0].sum()
        t.cuda.synchronize()
        for (_, out, _), want in zip(graphs, eager):
            for name in want:
                assert t.equal(out[name], want[name]), (i, name)
                out[name].zero_()
        t.cuda.synchronize()
    # new logits in the same buffer
    sets[0][0].copy_(t.randn(sets[0][0].shape, generator=g, device="cuda"))
    graphs[0][0].replay()
    want = TokenLogprobs().compute(*sets[0], top=7)
    t.cuda.synchronize()
    for name in want:
        assert t.equal(graphs[0][1][name], want[name]), name
    # another stream, waiting for the one that makes the logits
    x = t.randn(30, 20000, device="cuda")
    side.wait_stream(t.cuda.current_stream())
    got = TokenLogprobs().compute(x, top=5, stream=side)
    side.synchronize()
    want = TokenLogprobs().compute(x, top=5)
    for name in want:
        assert t.equal(got[name], want[name]), name


@pytest.mark.gpu
@pytest.mark.parametrize("rows,V", [(1, 40), (3, 33000), (70, 9000), (520, 2000)])
def test_memory_behind_the_rows_stays_as_it_was(torch_gpu, rows, V):
    from oxide_sampler import TokenLogprobs
    t = torch_gpu
    x = t.randn(rows, V, device="cuda")
    tokens = t.randint(0, V, (rows, 3), device="cuda", dtype=t.int32)
    shapes = {"logsumexp": (), "entropy": (), "status": (), "logprobs": (3,), "ranks": (3,), "top_ids": (4,),
              "top_logprobs": (4,)}
    whole = {n: t.full((rows + 2, *s), 77, dtype=t.int32 if n in ("status", "ranks", "top_ids") else t.float32,
                       device="cuda") for n, s in shapes.items()}
    lp = TokenLogprobs()
    lp.compute(x, tokens, top=4, out={n: w[1:rows + 1] for n, w in whole.items()})
    fresh = lp.compute(x, tokens, top=4)
    for n, w in whole.items():
        assert t.equal(w[1:rows + 1], fresh[n]), n
        assert bool((w[0] == 77).all()) and bool((w[rows + 1:] == 77).all()), n


@pytest.mark.gpu
def test_outputs_on_another_stream(torch_gpu):
    from oxide_sampler import TokenLogprobs
    t = torch_gpu
    x = t.randn(40, 50000, device="cuda")
    tokens = t.randint(0, 50000, (40,), device="cuda", dtype=t.int32)
    want = TokenLogprobs().compute(x, tokens, top=6)
    s = t.cuda.Stream()
    s.wait_stream(t.cuda.current_stream())
    lp = TokenLogprobs()
    outs = []
    for _ in range(5):
        junk = [t.zeros(40, device="cuda") for _ in range(3)]  # freed and reused on the current stream
        outs.append(lp.compute(x, tokens, top=6, stream=s))
        del junk
    s.synchronize()
    for o in outs:
        for n in want:
            assert t.equal(o[n], want[n]), n


@pytest.mark.gpu
def test_one_workspace_for_calls_of_all_sizes(torch_gpu):
    # rows split over workgroups in different ways, one call after the other on one workspace
    from oxide_sampler import TokenLogprobs
    lp, rng = TokenLogprobs(), np.random.default_rng(12)
    for rows, V, dtype, T, top in ((1, 262147, "f32", 3, 32), (300, 9001, "bf16", 1, 4), (2, 40000, "f32", 64, 0),
                                   (1, 70, "f32", 2, 8), (511, 3000, "f32", 1, 1), (33, 33000, "bf16", 2, 20),
                                   (1, 262147, "bf16", 1, 3)):
        x = wl.zipf_prior_logits(rng, min(rows, 3), V, 3.0)
        x = np.ascontiguousarray(x[np.arange(rows) % len(x)])
        x = bf16(x) if dtype == "bf16" else x
        tokens = some_tokens(x, T, rng)
        check(run(torch_gpu, x, tokens, top, dtype=dtype, lp=lp), reference(x, tokens, top), V,
              what=f"rows={rows} V={V}")


@pytest.mark.gpu
def test_python_refusals(torch_gpu):
    from oxide_sampler import TokenLogprobs
    t = torch_gpu
    lp = TokenLogprobs()
    x = t.zeros(2, 64, device="cuda")
    tok = t.zeros(2, 1, dtype=t.int32, device="cuda")
    bad = [
        lambda: lp.compute(x.cpu()), lambda: lp.compute(x.half()), lambda: lp.compute(x[0]),
        lambda: lp.compute(x.t()), lambda: lp.compute(x[:1].expand(2, 64)), lambda: lp.compute(x, tok.long()),
        lambda: lp.compute(x, tok[:1]), lambda: lp.compute(x, tok.cpu()), lambda: lp.compute(x, tok.expand(2, 65)),
        lambda: lp.compute(x, top=33), lambda: lp.compute(x, top=-1),
        lambda: lp.compute(x, mask=t.zeros(2, 1, dtype=t.int32, device="cuda")),
        lambda: lp.compute(x, mask=t.zeros(3, 2, dtype=t.int32, device="cuda")),
        lambda: lp.compute(x, temperatures=t.ones(3, device="cuda")),
        lambda: lp.compute(x, temperatures=t.ones(2, dtype=t.float64, device="cuda")),
        lambda: lp.compute(x, out={"entropy": t.zeros(2, 1, device="cuda")}),
        lambda: lp.compute(x, out={"status": t.zeros(2, device="cuda")}),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was taken")
    with pytest.raises(_abi.OxsError):
        lp.compute(x[:, :0])
    assert lp.compute(x[:0])["entropy"].shape == (0,)


@pytest.mark.gpu
def test_decode_loop_with_logprobs(torch_gpu):
    """The loop's tokens, states and events are those without log probabilities, captured or not, and each
    step's log probabilities are the definition's for its tokens."""
    from oxide_sampler import DecodeLoop
    t = torch_gpu
    S, V, rng = 6, 7001, np.random.default_rng(8)
    steps = [wl.zipf_prior_logits(rng, S, V, 3.0) for _ in range(5)]
    loops = [DecodeLoop(S, V, top_logprobs=n) for n in (None, 4, 0)]
    for loop in loops:
        for s in range(S - 1):  # one slot stays free
            loop.add_sequence(s, temperature=0.0 if s == 2 else 0.9, top_p=0.95, current_token=1,
                              current_position=3, max_tokens=50)
    buf = t.empty(S, V, device="cuda")
    mask = np.ones((S, V), bool)
    mask[1, 50:] = False
    words = t.from_numpy(wl.pack_mask(mask, V).view(np.int32)).cuda()
    for i, x in enumerate(steps):
        buf.copy_(t.from_numpy(x))
        if i == 2:
            loops[1].capture(buf, words)
        events = [loop.step() if loop is loops[1] and i >= 2 else loop.step(buf, words) for loop in loops]
        assert events[1] == events[0] and events[2] == events[0]
        t.cuda.synchronize()
        tokens = loops[0].out["tokens"].cpu().numpy()
        for loop, n in ((loops[1], 4), (loops[2], 0)):
            np.testing.assert_array_equal(loop.out["tokens"].cpu().numpy(), tokens)
            check({k: v.cpu().numpy() for k, v in loop.logprobs.items()},
                  reference(x, tokens[:, None], n, mask), V, what=f"step {i}")
    for s in range(S - 1):
        a, b = loops[0].state(s), loops[1].state(s)
        assert (a.generated_tokens, a.rng_state, a.mirostat_mu) == (b.generated_tokens, b.rng_state, b.mirostat_mu)
    with pytest.raises(ValueError):
        DecodeLoop(2, 100, top_logprobs=33)
    for loop in loops:
        loop.close()
