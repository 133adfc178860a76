"""What the entry points of speculative and sparse decoding refuse, without a GPU: fake CUDA tensors for the host module, null and
misfit parameters for the C ABI."""
import ctypes
import json
import os
import subprocess
import sys

import pytest

from test_host_checks_cpu import CACHE, CHILD, ROOT

B = "B = pikv_b200.PageBounds(t(8, 2, 2, 128, dtype=torch.int8), t(8, 2, dtype=f32)); "
TREE = CACHE + "q, m = t(4, 3, 8, 128), t(4, 3, 3, dtype=torch.bool); c.decode_attention_tree(%s)"
ACCEPT = CACHE + "c.accept_tree(%s)"
BOUNDS = CACHE + B + "c.update_bounds(%s)"
SPARSE = CACHE + B + "c.decode_attention_sparse(%s)"
CALLS = [
    (TREE % "q.float(), m", "BFloat16"),
    (TREE % "q[0], m", "must be [B, N, n_q"),
    (TREE % "t(4, 3, 8, 64), m", "must be [B, N, n_q"),
    (TREE % "torch.empty(4, 3, 8, 128, dtype=bf), m", "CUDA tensor"),
    (TREE % "q, None", "CUDA tensor"),
    (TREE % "q, m.int()", "Bool"),
    (TREE % "q, m[:, :2]", "mask must be"),
    (TREE % "q, m[:3]", "mask must be"),
    (TREE % "q, m[0, 0]", "mask must be"),
    (TREE % "t(5, 3, 8, 128), t(3, 3, dtype=torch.bool)", "5 streams, the cache has 4"),
    (TREE % "q, m, t(3, dtype=i32)", "are needed"),
    (TREE % "q, m, t(4, dtype=torch.int64)", "Int"),
    (TREE % "q, m, None, t(3, dtype=i32)", "are needed"),
    (TREE % "q, m, None, None, t(3, dtype=i32)", "are needed"),
    (TREE % "q, m, torch.empty(4, dtype=i32, device='cuda:1')", "different devices"),
    (ACCEPT % "t(4, dtype=i32)", "must be [B, depth]"),
    (ACCEPT % "t(4, 2)", "Int"),
    (ACCEPT % "t(5, 2, dtype=i32)", "5 streams, the cache has 4"),
    (ACCEPT % "t(4, 2, dtype=i32), t(3, dtype=i32)", "are needed"),
    (ACCEPT % "t(4, 2, dtype=i32), None, t(3, dtype=i32)", "are needed"),
    (ACCEPT % "t(4, 2, dtype=i32), None, None, t(2, dtype=i32)", "are needed"),
    (BOUNDS.replace("t(8, 2, dtype=f32)", "t(7, 2, dtype=f32)") % "B", "are needed"),
    (BOUNDS.replace("t(8, 2, 2, 128, dtype=torch.int8)", "t(8, 2, 128, dtype=torch.int8)") % "B", "are needed"),
    (BOUNDS.replace("t(8, 2, 2, 128, dtype=torch.int8)", "t(8, 2, 2, 256, dtype=torch.int8)[..., :128]") % "B", "must be contiguous"),
    (BOUNDS.replace("dtype=torch.int8", "dtype=torch.uint8") % "B", "Char"),
    (BOUNDS % "pikv_b200.PageBounds(None, None)", "must hold CUDA tensors"),
    (BOUNDS % "B, t(3, dtype=i32), t(2, dtype=i32)", "are needed"),
    (BOUNDS % "B, t(3, dtype=i32), None, t(2, dtype=i32)", "are needed"),
    (BOUNDS % "B, None, t(3, dtype=i32)", "are needed"),
    (SPARSE % "t(4, 8, 128), B, 0", "pages must be"),
    (SPARSE % "t(4, 8, 128), B, 1 << 20", "pages must be"),
    (SPARSE % "t(4, 8, 128), B, 4, first=-1", "must fit"),
    (SPARSE % "t(4, 8, 128), B, 4, recent=0", "must fit"),
    (SPARSE % "t(4, 8, 128), B, 4, first=2, recent=3", "must fit"),
    (SPARSE % "t(4, 8, 64), B, 4", "must be [B, n_q"),
    (SPARSE % "t(4, 8, 128).half(), B, 4", "BFloat16"),
    (SPARSE % "t(5, 8, 128), B, 4", "5 streams, the cache has 4"),
    (SPARSE % "t(4, 8, 128), B, 4, t(3, dtype=i32)", "are needed"),
    (SPARSE % "t(4, 8, 128), B, 4, None, t(3, dtype=i32)", "are needed"),
]


@pytest.fixture(scope="module")
def answers():
    r = subprocess.run([sys.executable, "-c", CHILD, json.dumps([c for c, _ in CALLS])], capture_output=True, text=True, cwd=ROOT,
                       env=dict(os.environ, PYTHONPATH=ROOT))
    assert r.returncode == 0, r.stderr[-2000:]
    return dict(json.loads(line) for line in r.stdout.splitlines())


@pytest.mark.parametrize("call,says", CALLS)
def test_refusals(answers, call, says):
    assert answers[call].startswith("PikvError: ") and says in answers[call], answers[call]


def test_abi_refusals():
    from pikv_b200 import _lib
    lib = _lib.lib()
    c = _lib.PagedCache()
    ref = ctypes.byref
    words = (ctypes.c_uint32 * 64)()
    at = (ctypes.addressof(words) + 15) & ~15                       # never read: every call is refused before a launch
    assert lib.pikv_tree_accept(ref(c), at, None, None, at, 1, 1, None, at, None) == -1 and b"null cache pointer" in lib.pikv_last_error()
    for f in ("page_table", "k_codes", "v_codes", "k_scale", "v_scale"):
        setattr(c, f, at)
    assert lib.pikv_page_bounds_update(ref(c), at, at, None, None, at, 1, None) == -1 and b"geometry" in lib.pikv_last_error()
    c.num_seqs, c.max_pages, c.num_pages, c.n_kv, c.bits, c.symmetric = 4, 8, 32, 2, 8, 0
    assert lib.pikv_page_bounds_update(ref(c), at, at, None, None, at, 1, None) == -2        # 8-bit asymmetric
    c.bits, c.symmetric = 4, 0
    assert lib.pikv_page_bounds_update(ref(c), at, at, None, None, at, 1, None) == -1 and b"k_zp" in lib.pikv_last_error()
    c.bits, c.symmetric = 8, 1
    c.k_codes = at + 8
    assert lib.pikv_page_bounds_update(ref(c), at, at, None, None, at, 1, None) == -1 and b"aligned" in lib.pikv_last_error()
    c.k_codes = at
    assert lib.pikv_page_bounds_update(ref(c), at, at, None, None, at, 5, None) == -1         # five streams of four
    assert lib.pikv_tree_accept(ref(c), at, None, None, at, 1, -1, None, at, None) == -1
    assert lib.pikv_tree_accept(ref(c), None, None, None, at, 1, 1, None, at, None) == -1
    assert lib.pikv_tree_accept(ref(c), at, None, at, at, 1, 1, at, at, None) == -1           # ctx_len is `length`, with ids

    t = _lib.TreeParams()
    t.q = t.out = t.ctx_len = t.mask = t.workspace = at
    t.B, t.N, t.n_q = 1, 65, 4
    assert lib.pikv_tree_attn(ref(c), ref(t), None) == -4 and b"nodes" in lib.pikv_last_error()
    t.N, t.n_q = 4, 3
    assert lib.pikv_tree_attn(ref(c), ref(t), None) == -1
    t.n_q = 130
    assert lib.pikv_tree_attn(ref(c), ref(t), None) == -2
    t.n_q, t.q = 4, at + 2
    assert lib.pikv_tree_attn(ref(c), ref(t), None) == -1 and b"aligned" in lib.pikv_last_error()
    assert lib.pikv_tree_attn_workspace_bytes(0, 4, 4, 2) == 0 and lib.pikv_tree_attn_workspace_bytes(2, 4, 4, 2) > 0

    s = _lib.SparseParams()
    s.q = s.out = s.seq_len = s.bound_codes = s.bound_scale = s.workspace = at
    s.B, s.n_q, s.pages, s.first, s.recent = 1, 4, 4, 3, 2
    assert lib.pikv_sparse_attn(ref(c), ref(s), None) == -1 and b"must fit" in lib.pikv_last_error()
    s.first, s.n_q = 0, 18
    assert lib.pikv_sparse_attn(ref(c), ref(s), None) == -2
    s.n_q = 4
    assert lib.pikv_sparse_attn(ref(c), ref(s), None) == -1 and b"workspace too small" in lib.pikv_last_error()
    c.max_pages = 50000
    assert lib.pikv_sparse_attn(ref(c), ref(s), None) == -4
    assert lib.pikv_sparse_attn_workspace_bytes(4, 8, 2, 64, 16) > lib.pikv_decode_attn_workspace_bytes(4, 8, 2, 0, 0)


def test_accept_overlapping_lengths():
    """A part of the lengths, or of the new ones, as an input: another stream's entry would be read while it is written."""
    from pikv_b200 import _lib
    lib = _lib.lib()
    words = (ctypes.c_uint32 * 64)()
    at = (ctypes.addressof(words) + 15) & ~15                       # never read: every call is refused before a launch
    c = _lib.PagedCache(page_table=at, num_seqs=4, max_pages=8, num_pages=32, n_kv=2, bits=8, symmetric=1, k_codes=at, v_codes=at, k_scale=at, v_scale=at)
    apart, length, new = at + 160, at + 64, at + 96                 # `length`: four words, `new`: two

    def call(path=apart, path_len=None, ids=None, ctx=apart, new_len=new):
        return lib.pikv_tree_accept(ctypes.byref(c), path, path_len, ids, ctx, 2, 2, length, new_len, None), lib.pikv_last_error()

    for over in (dict(ctx=length + 4), dict(ctx=length - 4), dict(ctx=length + 12, ids=apart), dict(ctx=new + 4), dict(ctx=new - 4), dict(path=length + 8),
                 dict(path=new - 12), dict(path_len=length), dict(path_len=new), dict(ids=length + 12), dict(ids=new), dict(new_len=length + 12)):
        rc, says = call(**over)
        assert rc == -1 and b"overlap" in says, over
