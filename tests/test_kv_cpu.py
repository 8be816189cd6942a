"""CPU suite of the KV cache: what the C ABI and the host mirror refuse, the reading of a call's
sequence lists (the kernels' own function, compiled for the host), and the reference's arithmetic."""
import ctypes as C
import os
import shutil
import subprocess

import numpy as np
import pytest
import torch

from tests import kv_reference as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")


@pytest.fixture(scope="module")
def lib():
    import huffman_amd
    return huffman_amd.lib()


def structs(**kw):
    from huffman_amd import _lib as L
    row = 128
    c = dict(d_k=4096, d_v=8192, d_k_scale=16384, d_v_scale=32768, n_pages=4, page_stride=16 * 8 * row,
             token_stride=8 * row, head_stride=row, page_size=16, heads=8, head_dim=128, group=128,
             format=L.HF_KV_FP8_E4M3, reserved=0)
    b = dict(d_cu_rows=0, d_kv_len=64, d_table=128, table_stride=4, table_width=4, batch=2, rows=2, max_rows=1)
    q = dict(d_q=4096, d_out=8192, d_lse=0, d_mask=0, q_row_stride=4096, q_head_stride=128,
             out_row_stride=4096, out_head_stride=128, q_heads=32, mask_words=0, dtype=L.HF_DT_BF16, scale=0.1)
    for k, v in kw.items():
        (c if k in c else b if k in b else q)[k] = v
    return L.hf_kv_cache(**c), L.hf_kv_batch(**b), L.hf_kv_query(**q)


ARG, ALIGN, RANGE = -1, -2, -3


def calls(lib, **kw):
    """Codes of the four calls without a context: -1 is what arguments in order give, too."""
    c, b, q = structs(**kw)
    c, b, q = C.byref(c), C.byref(b), C.byref(q)
    return (lib.hf_kv_write(None, c, b, 4096, 4096, 1024, 128, 1024, 128, 0),
            lib.hf_kv_read(None, c, b, 4096, 4096, 1024, 128, 1024, 128, 0),
            lib.hf_kv_attend(None, c, b, q, None, 0), lib.hf_kv_keep(None, c, b, 4096, 4, 4, 4096, 8192))


def test_no_context_no_structs(lib):
    assert calls(lib) == (ARG,) * 4
    assert lib.hf_kv_write(None, None, None, None, None, 0, 0, 0, 0, 0) == ARG
    assert lib.hf_kv_attend(None, None, None, None, None, 0) == ARG
    assert lib.hf_kv_attend_work_bytes(None, None, None, 8) == 0


@pytest.mark.parametrize("kw", [dict(d_k=4104), dict(d_v=8200), dict(d_k_scale=16392), dict(token_stride=1032),
                                dict(head_stride=136), dict(page_stride=16 * 1024 + 8)])
def test_misaligned_caches(lib, kw):
    assert calls(lib, **kw) == (ALIGN,) * 4


@pytest.mark.parametrize("kw", [dict(batch=1 << 31), dict(rows=1 << 31, d_cu_rows=64), dict(page_stride=1 << 32)])
def test_out_of_range(lib, kw):
    assert set(calls(lib, **kw)) == {RANGE}


def test_misaligned_rows(lib):
    c, b, q = structs()
    c, b = C.byref(c), C.byref(b)
    assert lib.hf_kv_write(None, c, b, 4100, 4096, 1024, 128, 1024, 128, 0) == ALIGN
    assert lib.hf_kv_write(None, c, b, 4096, 4096, 1028, 128, 1024, 128, 0) == ALIGN
    assert lib.hf_kv_read(None, c, b, 4096, 4096, 1024, 128, 1024, 130, 2) == ALIGN
    for kw in (dict(d_q=4098), dict(d_out=8200), dict(q_row_stride=4100), dict(out_head_stride=132)):
        assert lib.hf_kv_attend(None, c, b, C.byref(structs(**kw)[2]), None, 0) == ALIGN


def test_host_mirror_refuses_before_any_gpu():
    from huffman_amd import KvCache, HF_KV_BF16, HF_KV_FP4_E2M1, HF_KV_FP8_E4M3
    k = torch.zeros(4, 16, 8, 128, dtype=torch.uint8)
    s = torch.zeros(4, 8, 1, 16, dtype=torch.uint8)
    with pytest.raises(ValueError, match="device tensors"):
        KvCache(k, k, s, s)
    with pytest.raises(ValueError, match="format"):
        KvCache(k, k, s, s, fmt=9)
    with pytest.raises(ValueError, match="alike"):
        KvCache(k, k[:2], s, s)
    with pytest.raises(ValueError, match="alike"):
        KvCache(k, k.transpose(1, 2).contiguous().transpose(1, 2), s, s)
    with pytest.raises(TypeError):
        KvCache(k, k, fmt=HF_KV_BF16)
    with pytest.raises(TypeError):
        KvCache(k.view(torch.float8_e4m3fn), k.view(torch.float8_e4m3fn), s, s, fmt=HF_KV_FP4_E2M1)
    assert HF_KV_FP8_E4M3 == 2


SEQ_TEST = r'''
#include <cstdio>
#include <vector>
#include "hf_kv.h"
// every list of four offsets and two lengths out of a few values, against the rules written out
int main() {
    const int vals[] = {-2147483647 - 1, -1, 0, 1, 5, 9, 2147483647};
    const int lens[] = {-2147483647 - 1, -5, 0, 1, 8, 32, 33, 2147483647};
    long n = 0;
    for (int lo : vals) for (int hi : vals) for (int len : lens) for (int rows : {0, 5, 9})
        for (int most : {1, 9}) for (int width : {1, 2}) {
            int cu[3] = {0, lo, hi}, kv[2] = {0, len};
            hf_kv_seqs s{};
            s.cu = cu; s.kv_len = kv; s.width = width; s.batch = 2; s.rows = rows; s.most = most;
            const hf_kv_seq q = hf_kv_sequence(s, 1, 4);
            const long k = (long)hi - lo;
            const bool ok = lo >= 0 && hi >= lo && hi <= rows && k <= most && len >= k && len <= width * 16 && len >= 0;
            if (ok == q.bad) { printf("lo %d hi %d len %d rows %d most %d width %d\n", lo, hi, len, rows, most, width); return 1; }
            if (ok && (q.row0 != lo || q.n != k || q.len != len || q.past != len - k)) return 2;
            if (!ok && (q.row0 || q.n || q.len || q.past)) return 3;
            ++n;
        }
    printf("ok %ld\n", n);
}
'''


def test_sequence_lists_as_the_kernels_read_them(tmp_path):
    """The kernels take a sequence's place from hf_kv_sequence alone: lists that would lead outside
    the row tensors or the table give an empty sequence."""
    src, exe = tmp_path / "seq.hip", tmp_path / "seq"
    src.write_text(SEQ_TEST)
    if not shutil.which(HIPCC):
        pytest.skip("no hipcc")
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-O1", "-std=c++17", "-I", os.path.join(ROOT, "huffman_amd", "csrc"),
                    str(src), "-o", str(exe)], check=True, capture_output=True, timeout=300)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0 and out.stdout.startswith("ok"), (out.returncode, out.stdout)


def test_reference_rounding_against_torch():
    """The reference's codes of e4m3 and e5m2 are torch's casts of the scaled values."""
    rng = np.random.default_rng(3)
    x = (rng.standard_normal((200, 64)) * np.exp(3 * rng.standard_normal((200, 1)))).astype(np.float32).astype(np.float64)
    x[0] = 0
    x[1] = 448.0
    x[2, :8] = [0.0625, 0.09375, 0.03125, -0.03125, 1 / 512, 3 / 1024, 1 / 1024, 448]
    for fmt, dt in ((R.E4M3, torch.float8_e4m3fn), (R.E5M2, torch.float8_e5m2)):
        code, scale = R.quantise(x, fmt, 32)
        y = np.ldexp(x.reshape(200, 2, 32), 127 - scale.astype(int)[..., None])
        assert np.abs(y).max() <= R.LARGEST[fmt]
        assert (np.abs(y).max(-1) > R.LARGEST[fmt] / 2)[1:].all()
        want = torch.from_numpy(y.astype(np.float32)).to(dt).view(torch.uint8).numpy().reshape(200, 64)
        assert np.array_equal(code, want)


@pytest.mark.parametrize("fmt", [R.E4M3, R.E5M2, R.E2M1])
def test_reference_round_trip_is_within_half_a_step(fmt):
    rng = np.random.default_rng(4)
    x = rng.standard_normal((50, 64))
    code, scale = R.quantise(x, fmt, 32)
    y = R.dequantise(code, scale, fmt, 32)
    rel = {R.E4M3: 2.0 ** -4, R.E5M2: 2.0 ** -3, R.E2M1: 2.0 ** -2}[fmt]
    least = {R.E4M3: 2.0 ** -10, R.E5M2: 2.0 ** -17, R.E2M1: 0.25}[fmt]  # half of the smallest code
    step = np.ldexp(least, scale.astype(int) - 127)
    assert (np.abs(y - x) <= np.maximum(rel * np.abs(x), np.repeat(step, 32, -1)) * (1 + 1e-12)).all()
