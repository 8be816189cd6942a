"""CPU suite of the KV cache at its edges: what the kernels and the host mirror decide before they touch memory."""
import contextlib
import os
import shutil
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")


def run_on_host(tmp_path, source):
    """Builds a program over the kernels' header for the host and runs it."""
    if not shutil.which(HIPCC):
        pytest.skip("no hipcc")
    src, exe = tmp_path / "edge.hip", tmp_path / "edge"
    src.write_text(source)
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-O1", "-std=c++17", "-I", os.path.join(ROOT, "huffman_amd", "csrc"),
                    str(src), "-o", str(exe)], check=True, capture_output=True, timeout=300)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0 and out.stdout.startswith("ok"), (out.returncode, out.stdout)


PATH_TEST = r'''
#include <cstdio>
#include "hf_kv.h"
// every path of three steps out of a few values
int main() {
    const int vals[] = {-2147483647 - 1, -2147483647, -5, -3, -2, -1, 0, 1, 2, 7, 8, 9, 2147483647};
    long taken = 0;
    for (int a : vals) for (int b : vals) for (int c : vals) for (int n : {0, 1, 3, 8, 2147418112}) {
        const int path[3] = {a, b, c};
        bool all = true;
        for (int i = 0; i < 3; ++i) {
            const bool ok = hf_kv_path_ok(path, i, n);
            // a step that is taken names a row, whatever stands in front of it: its page is looked up
            if (ok && (path[i] < 0 || path[i] >= n)) { printf("step %d of %d %d %d, %d rows\n", i, a, b, c, n); return 1; }
            all = all && ok;
        }
        if (all != (0 <= a && a < b && b < c && c < n)) { printf("path %d %d %d, %d rows\n", a, b, c, n); return 2; }
        taken += all;
    }
    printf("ok %ld\n", taken);
}
'''


def test_steps_of_a_path_are_rows_whatever_stands_in_front(tmp_path):
    """Paths that ascend below zero: every step is judged by itself before the table is read for it."""
    run_on_host(tmp_path, PATH_TEST)


@pytest.mark.parametrize("shape", [(1, 16, 8, 128), (4, 16, 1, 128), (1, 16, 1, 128), (4, 1, 8, 128), (4, 16, 8, 128)])
@pytest.mark.parametrize("dtype,size", [(torch.uint8, 1), (torch.bfloat16, 2)])
def test_strides_of_pools(shape, dtype, size):
    """Dense pools have dense strides, whatever a dimension of one says; a stride of zero stays one."""
    from huffman_amd.kv import _pool_strides
    pages, tokens, heads, row = shape
    k = torch.zeros(shape, dtype=dtype)
    page, token, head = _pool_strides(k)
    row *= size
    assert (heads == 1 or head == row) and (tokens == 1 or token == heads * row) and (pages == 1 or page == tokens * heads * row)
    assert min(page, token, head) >= row  # what the calls ask for
    odd = k.as_strided(shape, [1 if n == 1 else s for n, s in zip(shape, k.stride())])
    assert _pool_strides(odd) == (page, token, head)
    for dim in range(3):
        if shape[dim] > 1:  # expanded along a dimension: its stride is refused, not replaced
            one = k.narrow(dim, 0, 1).expand(shape)
            assert one.stride(dim) == 0 and _pool_strides(one)[dim] == 0


ROWS_TEST = r'''
#include <cstdio>
#include <vector>
#include "hf_kv.h"
// strides from 0 to 40 of rows of 1, 3 and 4 elements, against every element counted
int main() {
    long touch = 0, apart = 0;
    for (int rows = 0; rows < 6; ++rows) for (int heads = 0; heads < 6; ++heads) for (int dim : {1, 3, 4})
        for (int rs = 0; rs <= 40; ++rs) for (int hs = 0; hs <= 40; ++hs) {
            std::vector<char> hit(6 * 40 * 2 + 8);
            bool want = false;
            for (int i = 0; i < rows; ++i) for (int j = 0; j < heads; ++j) for (int d = 0; d < dim; ++d)
                want = hit[i * rs + j * hs + d]++ || want;
            if (hf_kv_rows_touch(rows, heads, rs, hs, dim) != want) {
                printf("rows %d heads %d strides %d %d dim %d\n", rows, heads, rs, hs, dim);
                return 1;
            }
            ++(want ? touch : apart);
        }
    printf("ok %ld %ld\n", touch, apart);
}
'''


def test_rows_that_lie_on_one_another(tmp_path):
    run_on_host(tmp_path, ROWS_TEST)


@pytest.mark.parametrize("captured", [0, 1])
def test_the_pools_device_is_asked_for_a_capture(monkeypatch, captured):
    """Pools on the second device, the first one current: a stream without a context is refused if the pools'
    device records a capture on it, and only then."""
    from huffman_amd import api, kv
    now = [0]

    @contextlib.contextmanager
    def device(index):
        was, now[0] = now[0], index
        yield
        now[0] = was

    monkeypatch.setattr(api, "_default_ctx", {})
    monkeypatch.setattr(kv, "_raw_stream", lambda index: 77)
    monkeypatch.setattr(kv, "Context", lambda index, stream: ("context", index, stream))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda index: ("stream", index))
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: now[0] == captured)
    c = kv.KvCache.__new__(kv.KvCache)
    c._ctx, c._index = None, 1
    if captured == 1:
        with pytest.raises(RuntimeError, match="capture"):
            c.ctx
        assert api._default_ctx == {}
    else:
        assert c.ctx == ("context", 1, ("stream", 1)) and list(api._default_ctx) == [(1, 77)]
    assert now == [0]


MEET_TEST = r'''
#include <cstdio>
#include <cstring>
#include "hf_kv.h"
// two tensors of the same strides, moved against one another, against every element counted
int main() {
    long meet = 0, apart = 0;
    for (int rows = 0; rows < 5; ++rows) for (int heads = 0; heads < 5; ++heads) for (int dim : {1, 3, 4})
        for (int rs = 0; rs <= 24; ++rs) for (int hs = 0; hs <= 24; ++hs) {
            char hit[256];
            memset(hit, 0, sizeof hit);
            for (int i = 0; i < rows; ++i) for (int j = 0; j < heads; ++j) memset(hit + i * rs + j * hs, 1, dim);
            for (int off = -210; off <= 210; ++off) {
                bool want = false;
                for (int i = 0; i < rows; ++i) for (int j = 0; j < heads; ++j) for (int d = 0; d < dim; ++d) {
                    const int at = i * rs + j * hs + d + off;
                    want = want || (at >= 0 && at < 256 && hit[at]);
                }
                if (hf_kv_rows_meet(rows, heads, rs, hs, dim, off) != want) {
                    printf("rows %d heads %d strides %d %d dim %d apart %d\n", rows, heads, rs, hs, dim, off);
                    return 1;
                }
                ++(want ? meet : apart);
            }
        }
    printf("ok %ld %ld\n", meet, apart);
}
'''


def test_row_tensors_that_share_elements(tmp_path):
    run_on_host(tmp_path, MEET_TEST)
