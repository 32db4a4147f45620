"""Attention over the 4-bit paged cache against 64 bits, within what its kernels round (no
16-bit keys, queries or values, weights once to fp16): elementwise and row by row."""
import pytest

import kv4_tight as T
from test_kv4_gpu import BF, CHUNKS, DECODE, FP, _run, _setup

pytestmark = pytest.mark.gpu


def _check(dip, dtype, lens, qs, H, hkv, D, P, causal=True, q_scale=1.0):
    q, cache, table, cu = _setup(sum(lens) + 3 * H, lens, qs, H, hkv, D, P, dtype, q_scale=q_scale)
    out, lse = _run(dip, q, cache, table, lens, cu, causal=causal)
    step = max(1, cu[-1] // 40)
    picks = sorted(set(range(0, cu[-1], step)) | {cu[-1] - 1})
    picks = [t for t in picks if lens[max(r for r in range(len(lens)) if cu[r] <= t)] > 0]
    if not picks:
        return
    ref = T.rows(q.cuda(), cache.cuda(), table.cuda(), lens, cu, P, dtype, picks, causal)
    T.check(out[picks], lse[picks], ref, dtype)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("lens,H,hkv,D,P", DECODE + [([20000, 9000], 8, 2, 128, 64), ([50000], 4, 1, 64, 16)])
@pytest.mark.parametrize("q_scale", [1.0, 3.0, 12.0])
def test_decode(dip, dtype, lens, H, hkv, D, P, q_scale):
    _check(dip, dtype, lens, [1] * len(lens), H, hkv, D, P, q_scale=q_scale)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("lens,qs,H,hkv,D,P", CHUNKS + [([9000, 300], [700, 90], 8, 2, 128, 64),
                                                        ([6000], [3000], 16, 4, 64, 32)])
def test_chunks(dip, dtype, causal, lens, qs, H, hkv, D, P):
    for q_scale in (1.0, 3.0, 12.0):
        _check(dip, dtype, lens, qs, H, hkv, D, P, causal, q_scale)
