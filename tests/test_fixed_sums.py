"""The fixed predictors' error sums are plain sums over every sample, whatever the width and the block length: the oracle against
numpy's exact integers, the corpus seeds whose chunk holds an unpinned one, and the compiled kernels against the oracle on the
emulator (tests/emu)."""
import hashlib
import os
import subprocess
import sys

import numpy as np
import pytest

from oracle import oracle as O
from pyflac_amd import synth
from tests import cases, fuzzgen

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CHUNKS = sorted({s // 40 for s in cases.UNPINNED_FUZZ_SEEDS})


def exact_sums(x, sbps):
    """Sums of |k-th difference| over the samples from the fifth on; from 28 bits on every position that has a k-th difference."""
    x = [int(v) for v in x]
    tot = []
    d = x
    for k in range(5):
        tot.append(sum(abs(v) for v in d[0 if sbps >= 28 else 4 - k:]))
        d = [b - a for a, b in zip(d, d[1:])]
    return tot


@pytest.mark.parametrize('bps', range(17, 33))
@pytest.mark.parametrize('n', [5, 6, 7, 8, 9, 10, 11, 42, 66, 139, 510, 1932, 1933, 1934, 1935, 4095, 4096, 4097])
def test_oracle_sums_are_exact(bps, n):
    rng = np.random.default_rng(bps * 10000 + n)
    lim = 1 << (bps - 1)
    for kind in range(3):
        if kind == 0:
            x = rng.integers(-lim, lim, (n, 2))
        elif kind == 1:                                        # full-scale alternation: the largest sums there are
            x = np.where(np.arange(n)[:, None] % 2 == 0, lim - 1, -lim) * np.array([[1, -1]])
            x = np.clip(x, -lim, lim - 1)
        else:
            x = np.cumsum(rng.integers(-lim // 512 - 1, lim // 512 + 2, (n, 2)), axis=0)
            x = (x + lim) % (2 * lim) - lim
        cfg, rc = O.config(5, 2, bps, 48000, max(16, n), False)
        assert rc == 0
        _b, info = O.encode_frame(cfg, np.ascontiguousarray(x.astype(np.int32)), 0, want_info=True)
        x = x.astype(np.int64)
        sig = [x[:, 0], x[:, 1], (x[:, 0] + x[:, 1]) >> 1, x[:, 0] - x[:, 1]]
        assert info.n_candidates == 4
        for c, s in enumerate(sig):
            w, sb = info.cand[c].wasted, info.cand[c].sbps
            assert list(info.cand[c].fixed_tot) == exact_sums(s >> w, sb), (kind, c, w, sb)


@pytest.mark.parametrize('seed', [s for c in CHUNKS for s in range(c * 40, c * 40 + 40)])
def test_seed_bytes_match_the_recorded_ones(seed, fuzz_golden):
    if seed in cases.UNPINNED_FUZZ_SEEDS:
        pytest.skip(cases.UNPINNED_REASON)
    g, c = fuzz_golden[str(seed)], fuzzgen.case(seed)
    a32 = np.ascontiguousarray(c['pcm'].astype(np.int32))
    assert synth.pcm_hash(a32) == g['pcm_hash']
    cfg, rc = O.config(c['level'], c['ch'], c['bps'], c['sr'], c['bs'], c['subset'])
    assert rc == g['init_status']
    if rc:
        return
    cfg.limit_min_bitrate = 1 if c['limit_min_bitrate'] else 0
    stream, _ = O.encode_stream(cfg, a32)
    assert len(stream) == g['total_bytes'] and hashlib.sha256(stream).hexdigest() == g['sha256']
    out, res = O.decode_stream(stream)
    assert res.n_errors == 0 and np.array_equal(out, a32.reshape(out.shape))


@pytest.mark.parametrize('seed', sorted(cases.UNPINNED_FUZZ_SEEDS))
def test_unpinned_seeds_are_valid_and_lossless(seed, fuzz_golden):
    """Every CRC holds, every sample comes back, and the frames lie where the sizes say."""
    g, c = fuzz_golden[str(seed)], fuzzgen.case(seed)
    a32 = np.ascontiguousarray(c['pcm'].astype(np.int32))
    assert synth.pcm_hash(a32) == g['pcm_hash'] and g['total_bytes'] == cases.UNPINNED_FUZZ_SEEDS[seed][0]
    cfg, rc = O.config(c['level'], c['ch'], c['bps'], c['sr'], c['bs'], c['subset'])
    assert rc == g['init_status'] == 0
    cfg.limit_min_bitrate = 1 if c['limit_min_bitrate'] else 0
    stream, sizes = O.encode_stream(cfg, a32)
    head = len(stream) - int(sizes.sum())
    for off, size in zip(head + np.concatenate([[0], np.cumsum(sizes)[:-1]]), sizes):
        f = np.frombuffer(stream[int(off):int(off) + int(size)], np.uint8)
        assert O.lib().flo_crc16(np.ascontiguousarray(f).ctypes.data, len(f)) == 0       # (a frame with its CRC-16 leaves no rest)
    out, res = O.decode_stream(stream)
    assert res.n_errors == 0 and np.array_equal(out, a32.reshape(out.shape))


@pytest.mark.skipif(not os.path.exists('/opt/rocm/lib/llvm/bin/llvm-objdump'), reason='the emulator reads the code objects through llvm-objdump')
def test_compiled_kernels_against_the_oracle_on_the_emulator():
    p = subprocess.run([sys.executable, '-m', 'pytest', '-q', '-x', '-p', 'tests.emu.plugin', '-m', 'gpu', '-k', 'not recorded_ones', 'tests/test_gpu_fixed_sums.py'],
                       capture_output=True, text=True, timeout=550, cwd=ROOT)
    assert p.returncode == 0 and ' failed' not in p.stdout, (p.stdout[-3000:], p.stderr[-2000:])
