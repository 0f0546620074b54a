"""The serving step's entry points without a device: what they refuse, and the
descriptors' layouts against the header's."""
import ctypes as C
import os
import re
import subprocess

import pytest

import warp_b200 as wb
from warp_b200 import build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
A = 1 << 20                                        # an address that no call may touch


@pytest.fixture(scope="module")
def lib():
    build.build()
    return wb.load_library()


def plan(**kw):
    p = {n: A + 64 * i for i, (n, t) in enumerate(wb.KvPlan._fields_) if t is C.c_void_p}
    return wb.KvPlan(**{**dict(B=2, T=4, page=16, max_blocks=8, n_free=4, mask_words=1), **p, **kw})


def rows(**kw):
    p = {n: A + 64 * i for i, (n, t) in enumerate(wb.MlaRows._fields_) if t is C.c_void_p}
    return wb.MlaRows(**{**dict(T=4, kl=512, rope=64, x_dtype=0, dtype=2, x_stride=576, row_stride=576, n_rows=64,
                                eps=1e-6), **p, **kw})


def tree(**kw):
    p = {n: A + 256 * i for i, (n, t) in enumerate(wb.MlaTree._fields_) if t is C.c_void_p}
    return wb.MlaTree(**{**dict(B=2, T=4, heads=32, kl=512, rope=64, dtype=2, page=16, max_blocks=8, mask_words=1,
                                n_blocks=32, row_stride=576, q_token_stride=32 * 576, q_head_stride=576,
                                o_token_stride=32 * 512, o_head_stride=512, scale=0.1, ws_bytes=1 << 40), **p, **kw})


def logits(**kw):
    p = {n: A + 64 * i for i, (n, t) in enumerate(wb.LogitsAdjust._fields_) if t is C.c_void_p}
    return wb.LogitsAdjust(**{**dict(B=2, R=4, V=1000, dtype=0, tree_words=1, allow_words=32, n_allow=4,
                                     hist_stride=16, ld=1000, ld_out=1000), **p, "out": A + (1 << 16), **kw})


REFUSED = [
    ("kv_plan_dev", plan, dict(B=0)), ("kv_plan_dev", plan, dict(B=4097)), ("kv_plan_dev", plan, dict(T=-1)),
    ("kv_plan_dev", plan, dict(page=0)), ("kv_plan_dev", plan, dict(max_blocks=0)),
    ("kv_plan_dev", plan, dict(page=1 << 16, max_blocks=1 << 16)), ("kv_plan_dev", plan, dict(n_free=-1)),
    ("kv_plan_dev", plan, dict(free_blocks=None)), ("kv_plan_dev", plan, dict(ctx_len=None)),
    ("kv_plan_dev", plan, dict(slot=None)), ("kv_plan_dev", plan, dict(short_blocks=None)),
    ("kv_plan_dev", plan, dict(mask=None)), ("kv_plan_dev", plan, dict(mask_words=0)),
    ("kv_plan_dev", plan, dict(kv_len=A, ctx_len=A)), ("kv_plan_dev", plan, dict(slot=A + 4)),
    ("kv_plan_dev", plan, dict(n_blocks=A, n_blocks_out=A + 4)), ("kv_plan_dev", plan, dict(n_blocks=A, kv_len=A)),
    ("kv_plan_dev", plan, dict(q_len=A + 8, q_indptr=A)),
    ("mla_rows_dev", rows, dict(T=-1)), ("mla_rows_dev", rows, dict(kl=0)), ("mla_rows_dev", rows, dict(kl=4097)),
    ("mla_rows_dev", rows, dict(rope=63)), ("mla_rows_dev", rows, dict(rope=514)),
    ("mla_rows_dev", rows, dict(dtype=3)), ("mla_rows_dev", rows, dict(x_dtype=-1)),
    ("mla_rows_dev", rows, dict(x_stride=575)), ("mla_rows_dev", rows, dict(row_stride=575)),
    ("mla_rows_dev", rows, dict(eps=float("nan"))), ("mla_rows_dev", rows, dict(slot=None)),
    ("mla_rows_dev", rows, dict(pos=None)), ("mla_rows_dev", rows, dict(cache=A + 1)),
    ("mla_tree_attn_dev", tree, dict(heads=0)), ("mla_tree_attn_dev", tree, dict(kl=513)),
    ("mla_tree_attn_dev", tree, dict(rope=129)), ("mla_tree_attn_dev", tree, dict(dtype=7)),
    ("mla_tree_attn_dev", tree, dict(page=0)), ("mla_tree_attn_dev", tree, dict(page=1 << 20, max_blocks=1 << 12)),
    ("mla_tree_attn_dev", tree, dict(T=1 << 30)), ("mla_tree_attn_dev", tree, dict(row_stride=512)),
    ("mla_tree_attn_dev", tree, dict(q_head_stride=512)), ("mla_tree_attn_dev", tree, dict(o_head_stride=511)),
    ("mla_tree_attn_dev", tree, dict(scale=float("inf"))), ("mla_tree_attn_dev", tree, dict(scale=float("nan"))),
    ("mla_tree_attn_dev", tree, dict(mask_words=0)), ("mla_tree_attn_dev", tree, dict(ws=A + 16)),
    ("mla_tree_attn_dev", tree, dict(q=None)), ("mla_tree_attn_dev", tree, dict(o=A + 1)),
    ("mla_tree_attn_dev", tree, dict(o=A, q=A)),
    ("logits_adjust_dev", logits, dict(V=0)), ("logits_adjust_dev", logits, dict(B=4097)),
    ("logits_adjust_dev", logits, dict(R=65536)), ("logits_adjust_dev", logits, dict(logits=A, out=A + 400)),
    ("logits_adjust_dev", logits, dict(ld=999)), ("logits_adjust_dev", logits, dict(ld_out=999)),
    ("logits_adjust_dev", logits, dict(dtype=3)), ("logits_adjust_dev", logits, dict(q_indptr=None)),
    ("logits_adjust_dev", logits, dict(hist_len=None)), ("logits_adjust_dev", logits, dict(draft=None)),
    ("logits_adjust_dev", logits, dict(tree_words=0)), ("logits_adjust_dev", logits, dict(bias_val=None)),
    ("logits_adjust_dev", logits, dict(allow_words=31)), ("logits_adjust_dev", logits, dict(logits=A, out=A, ld_out=1004)),
    ("logits_adjust_dev", logits, dict(out=A + 2)),
    ("kv_plan_dev", plan, dict(pos=A, ctx_len=A)), ("kv_plan_dev", plan, dict(slot=A + 8, q_len=A + 36)),
    ("kv_plan_dev", plan, dict(mask=A, parent=A + 12)), ("kv_plan_dev", plan, dict(block_table=A, free_blocks=A + 60)),
    ("kv_plan_dev", plan, dict(short_blocks=A, free_head=A)), ("kv_plan_dev", plan, dict(free_head_out=A + 4, n_blocks=A)),
    ("kv_plan_dev", plan, dict(pos=A, slot=A)), ("kv_plan_dev", plan, dict(n_blocks_out=A, kv_len=A)),
    ("kv_plan_dev", plan, dict(mask_words=1 << 26)), ("mla_tree_attn_dev", tree, dict(mask_words=1 << 26)),
    ("logits_adjust_dev", logits, dict(tree_words=1 << 26)),
    ("mla_tree_attn_dev", tree, dict(o_token_stride=512)), ("mla_tree_attn_dev", tree, dict(o_token_stride=1024)),
    ("mla_tree_attn_dev", tree, dict(o_token_stride=512 * 31 + 511)), ("mla_tree_attn_dev", tree, dict(o_token_stride=700, o_head_stride=1000)),
    ("mla_tree_attn_dev", tree, dict(o_token_stride=512, o_head_stride=512 * 4 - 1)),
    ("mla_tree_attn_dev", tree, dict(T=(1 << 20) + 1)), ("mla_tree_attn_dev", tree, dict(T=1 << 19, max_blocks=1 << 13)),
    ("mla_tree_attn_dev", tree, dict(B=1 << 28, max_blocks=1 << 9)),
]


@pytest.mark.parametrize("name,make,wrong", REFUSED,
                         ids=[f"{n}-{'-'.join(w)}-{i}" for i, (n, _, w) in enumerate(REFUSED)])
def test_refused(lib, name, make, wrong):
    with pytest.raises(wb.WasteCudaError) as e:
        getattr(wb, name)(make(**wrong))
    assert e.value.rc == wb.E_ARG and name in str(e.value)


@pytest.mark.parametrize("ts,hs,T,heads", [(512 * 32, 512, 4, 32), (512, 512 * 4, 4, 32), (512 * 31 + 512, 512, 4, 32),
                                           (520, 4 * 520 - 8, 4, 32), (1024, 1024 * 4 + 512, 4, 32), (512, 512, 1, 32),
                                           (512, 512, 4, 1), (1024, 1536, 2, 2), (1 << 62, 1 << 57, 4, 32)])
def test_attn_rows_apart(lib, ts, hs, T, heads):
    """Layouts of o whose rows share nothing pass the checks (and ask for a device)."""
    if wb.load_library().waste_cuda_device() >= 0:
        pytest.skip("another test bound the library")
    with pytest.raises(wb.WasteCudaError) as e:
        wb.mla_tree_attn_dev(tree(o_token_stride=ts, o_head_stride=hs, T=T, heads=heads))
    taken = sorted(t * ts + h * hs for t in range(T) for h in range(heads))
    assert all(b - a >= 512 for a, b in zip(taken, taken[1:]))
    assert e.value.rc == wb.E_NODEV


def test_attn_limits(lib):
    """The largest sizes the header allows pass the checks, one more is refused
    with the numbers."""
    if wb.load_library().waste_cuda_device() >= 0:
        pytest.skip("another test bound the library")
    units = lambda T, heads, B, cols, page: (T * heads // 32 + B + 1) * (page * cols // 32 + 2)
    cols = next(c for c in range(1, 1 << 20) if units(64, 32, 2, c + 1, 1 << 11) >= 1 << 31)
    for kw in (dict(T=1 << 20), dict(T=64, max_blocks=cols, page=1 << 11)):
        with pytest.raises(wb.WasteCudaError) as e:
            wb.mla_tree_attn_dev(tree(**kw))
        assert e.value.rc == wb.E_NODEV, kw
    with pytest.raises(wb.WasteCudaError) as e:
        wb.mla_tree_attn_dev(tree(T=64, max_blocks=cols + 1, page=1 << 11))
    assert e.value.rc == wb.E_ARG and str(units(64, 32, 2, cols + 1, 1 << 11)) in str(e.value)


def test_null_descriptors(lib):
    for n in ("kv_plan_dev", "mla_rows_dev", "mla_tree_attn_dev", "logits_adjust_dev"):
        assert getattr(lib, "waste_cuda_" + n)(None, None) == wb.E_ARG


def test_plan_counts_in_place(lib):
    """What the counts may share passes the checks (and asks for a device)."""
    if wb.load_library().waste_cuda_device() >= 0:
        pytest.skip("another test bound the library")
    for kw in (dict(n_blocks=A, n_blocks_out=A), dict(free_head=A, free_head_out=A), dict(T=0, pos=A, ctx_len=A),
               dict(n_free=0, free_blocks=A, kv_len=A)):
        with pytest.raises(wb.WasteCudaError) as e:
            wb.kv_plan_dev(plan(**kw))
        assert e.value.rc == wb.E_NODEV, kw


def test_nothing_to_do(lib):
    """No tokens, rows or requests: done without a device."""
    wb.mla_rows_dev(rows(T=0))
    wb.mla_tree_attn_dev(tree(T=0))
    wb.mla_tree_attn_dev(tree(B=0))
    wb.logits_adjust_dev(logits(R=0))


def test_workspace_sizes_out_of_range(lib):
    assert wb.mla_tree_ws_bytes(0, 512) == 0
    assert wb.mla_tree_ws_bytes(32, 513) == 0


def test_before_init(lib):
    """With no library bound, every call says so (and touches nothing)."""
    if wb.load_library().waste_cuda_device() >= 0:
        pytest.skip("another test bound the library")
    for f, d in ((wb.kv_plan_dev, plan()), (wb.mla_rows_dev, rows()), (wb.mla_tree_attn_dev, tree()),
                 (wb.logits_adjust_dev, logits())):
        with pytest.raises(wb.WasteCudaError) as e:
            f(d)
        assert e.value.rc == wb.E_NODEV


@pytest.mark.parametrize("cls,name", [(wb.KvPlan, "waste_cuda_kv_plan_desc"), (wb.MlaRows, "waste_cuda_mla_rows_desc"),
                                      (wb.MlaTree, "waste_cuda_mla_tree_desc"),
                                      (wb.LogitsAdjust, "waste_cuda_logits_desc")])
def test_descriptor_layout(tmp_path, cls, name):
    """Sizes and offsets of the ctypes mirrors are the C compiler's."""
    src = tmp_path / "s.c"
    lines = [f'printf("%zu\\n", sizeof({name}));'] + \
            [f'printf("%zu\\n", offsetof({name}, {f[0]}));' for f in cls._fields_]
    src.write_text('#include <stdio.h>\n#include "waste_cuda.h"\nint main(void){%s return 0;}' % "".join(lines))
    exe = tmp_path / "s"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), "-o", str(exe), str(src)], check=True)
    out = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert out == [C.sizeof(cls)] + [getattr(cls, f[0]).offset for f in cls._fields_]
    body = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "waste_cuda.h")).read(), flags=re.S)
    body = body[:body.index("} " + name)]
    names = re.findall(r"\w+(?=\s*[,;])", body[body.rindex("typedef struct {"):])
    assert names == [f[0] for f in cls._fields_]
