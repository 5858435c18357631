"""CPU-side checks of the paged 8-bit cache's operators: argument errors of the
C ABI come before any device work, workspace sizes are host-only, the torch
binding refuses CPU tensors, and the tests' plain forms agree with torch."""
import math

import pytest
import torch

import paged_ref as ref
import pmkl_b200

FAKE = 0x10000  # non-null, 256-byte aligned, never dereferenced


def plan(batch=2, max_blocks=4, block=16, tokens=8, stride=4, cap=3, ptr=FAKE, out=0x20000):
    return pmkl_b200.capi().pmkl_paged_plan(ptr, ptr, ptr, stride, ptr, ptr, cap, batch, max_blocks, block, tokens, ptr,
                                            ptr, ptr, out, ptr, None)


def test_plan_argument_errors():
    assert plan(batch=-1) == -1
    assert plan(block=0) == -1
    assert plan(tokens=-1) == -1
    assert plan(tokens=1 << 31) == -1
    assert plan(stride=3) == -1  # rows overlap
    assert plan(out=FAKE) == -1  # free_count_out is free_count
    assert plan(ptr=0) == -3
    assert plan(out=0) == -3


def append(tokens=2, heads=1, hidden=64, dtype=2, blocks=4, block=16, ptr=FAKE, strides=None):
    return pmkl_b200.capi().pmkl_paged_append(ptr, ptr, strides, None, ptr, tokens, heads, hidden, dtype, ptr, ptr, None,
                                              None, ptr, ptr, blocks, block, None)


def test_append_argument_errors():
    import ctypes
    assert append(tokens=-1) == -1
    assert append(block=0) == -1
    assert append(dtype=7) == -2
    assert append(hidden=257) == -5
    assert append(ptr=0) == -3
    assert append(strides=(ctypes.c_int64 * 2)(-1, 64)) == -1
    assert append(tokens=0, ptr=0) == 0 and append(blocks=0, ptr=0) == 0


def attend(tokens=2, batch=2, heads=4, kv=2, hidden=64, blocks=4, block=16, width=4, stride=4, max_q=1, dtype=2, kernel=0,
           ptr=FAKE, starts=FAKE, ws=FAKE, ws_bytes=1 << 40):
    return pmkl_b200.capi().pmkl_paged_attention(ptr, None, ptr, ptr, None, None, ptr, ptr, ptr, stride, ptr, starts, ptr,
                                                 None, ptr, tokens, batch, heads, kv, hidden, blocks, block, width, max_q,
                                                 dtype, 1, 0.0, ws, ws_bytes, kernel, None)


def test_attention_argument_errors():
    assert attend(tokens=-1) == -1
    assert attend(kv=3) == -1
    assert attend(kv=0) == -1
    assert attend(stride=3) == -1
    assert attend(tokens=3, starts=None) == -1  # one token a request
    assert attend(block=0) == -1
    assert attend(max_q=0x7FFFFFFF, heads=8, kv=1) == -1  # rows of a K/V head past 31 bits
    assert attend(dtype=5) == -2
    assert attend(kernel=77) == -5
    assert attend(hidden=257) == -5
    assert attend(ptr=0) == -3
    assert attend(tokens=0, ptr=0, batch=0) == 0


def test_workspace_size_is_zero_for_empty_or_bad_sizes():
    f = pmkl_b200.capi().pmkl_paged_attention_workspace_size
    assert f(0, 2, 4, 2, 64, 1, 2) == 0
    assert f(2, 2, 4, 3, 64, 1, 2) == 0
    assert f(2, 2, 4, 2, 64, 1, 9) == 0
    assert f(2, 2, 4, 2, 64, 1, 2) % 256 == 0


@pytest.mark.parametrize("hidden", [64, 128])
@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_workspace_is_asked_for_whatever_max_query_len(hidden, dtype):
    """Without query_starts a request has one token, and the workspace of one, also where max_query_len says 0."""
    f = pmkl_b200.capi().pmkl_paged_attention_workspace_size_ex
    need = f(2, 2, 4, 2, hidden, 1, dtype, 0)
    assert need > 0 and f(2, 2, 4, 2, hidden, 0, dtype, 0) == need
    for max_q in (0, 1):
        for starts in (None, FAKE):
            assert attend(hidden=hidden, dtype=dtype, max_q=max_q, starts=starts, ws=None, ws_bytes=0) == -3
            assert attend(hidden=hidden, dtype=dtype, max_q=max_q, starts=starts, ws_bytes=need - 1) == -9
    # an upper limit far above the one token is no reason to refuse
    assert attend(hidden=hidden, dtype=dtype, heads=8, kv=1, max_q=0x7FFFFFFF, starts=None, ws=None) == -3


@pytest.mark.parametrize("hidden", [64, 128])
@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_workspace_size_goes_by_the_kernel(hidden, dtype):
    """A decode step asks for no more than its kernel can use: of 640 CTAs a descriptor and twice 8 rows with their sums."""
    import ctypes

    L = pmkl_b200.capi()
    size = lambda max_q, kernel, tokens=64: L.pmkl_paged_attention_workspace_size_ex(  # noqa: E731
        tokens, 64, 8, 2, hidden, max_q, dtype, kernel)
    rows = lambda ctas, n: -(-ctas * (32 + 2 * n * (hidden + 1) * 4) // 256) * 256  # noqa: E731
    assert size(1, 0) == size(1, 2) == rows(640, 8) and size(8, 2) == rows(640, 32)
    assert size(1, 1) == 0
    any_of = lambda max_q: L.pmkl_paged_attention_workspace_size(64, 64, 8, 2, hidden, max_q, dtype)  # noqa: E731
    if dtype:  # (tcgen05: 16-bit queries, from 33 rows a K/V head on)
        assert size(1, 3) == size(9, 0) == any_of(1) == any_of(9) == rows(320, 128) and size(8, 0) == rows(640, 32)
    else:
        assert size(9, 0) == size(9, 2) == any_of(9) == rows(640, 32)
    # What a call needs goes by its kernel.  Negative strides, which are looked at after the
    # workspace, end each call before anything is launched.
    bad = (ctypes.c_int64 * 2)(-1, -1)

    def call(kernel, ws, ws_bytes):
        return L.pmkl_paged_attention(FAKE, bad, FAKE, FAKE, None, None, FAKE, FAKE, FAKE, 4, FAKE, FAKE, FAKE, None, FAKE, 64, 64,
                                      8, 2, hidden, 4, 16, 4, 1, dtype, 1, 0.0, ws, ws_bytes, kernel, None)

    need = size(1, 0)
    assert call(0, FAKE, need) == -1 and call(0, FAKE, need - 1) == -9 and call(0, None, need) == -3
    assert call(1, None, 0) == -1
    if dtype:
        assert call(3, FAKE, need) == -9 and call(3, FAKE, size(1, 3)) == -1


def test_binding_refuses_cpu_tensors():
    from pmkl_function import paged_append, paged_attention, paged_plan

    n = torch.ones(1, dtype=torch.int32)
    c, s = torch.zeros(1, 1, 16, 64).to(torch.float8_e4m3fn), torch.ones(1, 1)
    x = torch.zeros(1, 1, 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged_attention(x, c, c, s, s, n[None], n)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged_append(x, x, torch.zeros(1, dtype=torch.int64), c, c, s, s)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged_plan(n, n, n[None], n, n, 16, 1)


def test_plain_forms():
    """The tests' own references: e4m3 rounding as torch's, attention as softmax of whole matrices."""
    x = torch.cat([torch.linspace(-500, 500, 4001), torch.linspace(-0.02, 0.02, 4001)]).double()
    assert torch.equal(ref.e4m3(x), x.float().clamp(-448, 448).to(torch.float8_e4m3fn).double())
    assert ref.scale_for(448.0) == 1 and ref.scale_for(448.1) == 2 and ref.scale_for(0) == 2.0 ** -64
    kc, ks = ref.make_cache(3, 1, 4, 8, 1)
    vc, vs = ref.make_cache(3, 1, 4, 8, 2)
    q = torch.randn(2, 2, 8, generator=torch.Generator().manual_seed(3))
    o, lse, _ = ref.attention(q, kc, vc, ks, vs, [[2, 0, 1]], [10], [0, 2])
    k = torch.cat([kc[p, 0].double() * ks[p, 0].double() for p in (2, 0, 1)])[:10]
    v = torch.cat([vc[p, 0].double() * vs[p, 0].double() for p in (2, 0, 1)])[:10]
    for i, keys in ((0, 9), (1, 10)):
        s = q[i, 1].double() @ k[:keys].T / math.sqrt(8)
        assert torch.allclose(o[i, 1], torch.softmax(s, 0) @ v[:keys]) and torch.allclose(lse[i, 1], s.logsumexp(0))
    seq, starts, slots, left, status, table = ref.plan([5, 0], [4, 2], [[7, 8, -1], [-1] * 3], [1, 2, 3], 3, 4, 7)
    assert (seq, starts, left, status) == ([9, 2], [0, 4, 6], 1, [0, 0])
    assert table == [[7, 8, 3], [2, -1, -1]] and slots == [33, 34, 35, 12, 8, 9, -1]


def test_walk_over_shares(tmp_path):
    """The device code that hands an attention's tiles out to CTAs, run on the host: every tile once, in order."""
    import subprocess
    from pathlib import Path

    from pmkl_b200 import build

    repo = Path(__file__).resolve().parent.parent
    exe = tmp_path / "walk_test"
    subprocess.run([build._nvcc(), *build.NVCC_ARCH, "-O1", "-std=c++17", "-I", str(build.INCLUDE), "-I", str(build.CSRC),
                    str(repo / "tests" / "cpp" / "walk_test.cu"), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0 and "walk ok" in out.stdout, out.stdout


def test_shares_of_long_lists(tmp_path):
    """Where the shares of more than 2^32 tiles begin, and whose a tile is."""
    import subprocess
    from pathlib import Path

    from pmkl_b200 import build

    repo = Path(__file__).resolve().parent.parent
    exe = tmp_path / "share_test"
    subprocess.run([build._nvcc(), *build.NVCC_ARCH, "-O1", "-std=c++17", "-I", str(build.INCLUDE), "-I", str(build.CSRC),
                    str(repo / "tests" / "cpp" / "share_test.cu"), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0 and "shares ok" in out.stdout, out.stdout
