"""Where the output of prompt attention may lie: the C entry refuses one that shares
rows with k, v or with other rows of q, before any launch (fake, never
dereferenced addresses), by a test of strided rows that a host program compares
with every byte (rows_meet_check.cpp)."""
import shutil
import subprocess
from pathlib import Path

import pytest

from nsn_amd import _lib

HERE = Path(__file__).resolve().parent
A, E = 1 << 20, _lib.NSN_EINVAL
N, HQ, HKV, ROW = 10, 8, 2, 256     # tokens, heads, bytes of a row
FAR = A + (1 << 30)


def test_rows_meet(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    exe = tmp_path / "rows_meet_check"
    subprocess.run([gxx, "-std=c++17", "-O1", "-Wall", "-o", str(exe), str(HERE / "rows_meet_check.cpp")], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0 and " 0 mismatches" in r.stdout, r.stdout


@pytest.mark.parametrize("where", [
    dict(out=A + ROW),                                           # other rows of q
    dict(out=A - N * HQ * ROW + 16),                             # its first 16 bytes
    dict(q=FAR + (1 << 26), k=A + N * HQ * ROW - 16, out=A),     # k in the output's last row
    dict(q=FAR + (1 << 26), v=A - N * HKV * ROW + 16, out=A),    # v's last row in the output's first
    dict(q=FAR + (1 << 26), k=A, out=A), dict(q=FAR + (1 << 26), v=A, out=A),
    dict(out=A, q_token_stride=HQ * 128 + 8), dict(out=A, q_head_stride=136),   # in place, but other rows
    dict(q=FAR + (1 << 26), k=A, k_token_stride=1 << 20, out=A + (1 << 21) - ROW),   # between k's rows, into the next
])
def test_an_output_among_the_inputs_is_refused(where):
    a = dict(q=A, k=FAR, v=FAR + (1 << 24), dtype=_lib.DTYPE_BF16, tokens=N, seqs=2, heads_q=HQ, heads_kv=HKV,
             q_token_stride=HQ * 128, q_head_stride=128, k_token_stride=HKV * 128, k_head_stride=128,
             v_token_stride=HKV * 128, v_head_stride=128, cu_seqlens=A, scale=0.1, out=FAR + (1 << 25), status=A)
    a.update(where)
    assert _lib.lib().nsn_prompt_attention(_lib.PromptArgs(**a), None) == E
