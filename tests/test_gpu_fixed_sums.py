"""The encoder's bytes against the oracle's where the block's length past the four warm-up samples takes every residue modulo four,
at 16 to 32 bits, in the pipeline and in the generic kernel; the recorded corpus seed by seed where its chunk holds an unpinned seed."""
import hashlib

import numpy as np
import pytest

from tests import cases, fuzzgen

pytestmark = pytest.mark.gpu
CHUNKS = sorted({s // 40 for s in cases.UNPINNED_FUZZ_SEEDS})


@pytest.fixture(scope='module')
def ctx():
    import torch
    from pyflac_amd import batch
    assert torch.cuda.is_available()
    return batch.Context(0)


@pytest.fixture(scope='module')
def hctx():
    from pyflac_amd import batch
    return batch.Context(0, testhooks=True)


def _check(ctx, pcm, ch, bps, level, bs, sr=48000, subset=False, lmb=False):
    import torch
    from pyflac_amd import batch
    from pyflac_amd.encoder import stream_header_bytes
    from oracle import oracle as O
    a = np.ascontiguousarray(np.asarray(pcm).reshape(-1, ch).astype(np.int32))
    s = batch.settings(level, ch, bps, sr, bs, subset)
    cfg, rc = O.config(level, ch, bps, sr, bs, subset)
    assert rc == 0
    s.limit_min_bitrate = cfg.limit_min_bitrate = 1 if lmb else 0
    t = torch.from_numpy(a).cuda()
    out, offs, st = ctx.encode(s, t)
    stream = stream_header_bytes(s) + out[:st.total_bytes].cpu().numpy().tobytes()
    want, sizes = O.encode_stream(cfg, a)
    assert [int(x) for x in np.diff(offs.cpu().numpy())] == [int(x) for x in sizes]
    assert stream == want
    dec, status, _ = ctx.decode(out[:st.total_bytes], offs, ch, bps, len(a))
    assert int(status[:, 0].max()) == 0 and torch.equal(dec.reshape(-1, ch), t)
    return stream


def _content(rng, n, ch, bps, kind):
    lim = 1 << (bps - 1)
    if kind == 0:                                              # a walk that wraps, with noise on it: orders 0 .. 4 lie close together
        x = np.cumsum(rng.integers(-lim // 64 - 1, lim // 64 + 2, (n, ch)), axis=0) + rng.integers(-lim // 4096 - 1, lim // 4096 + 2, (n, ch))
        return (x + lim) % (2 * lim) - lim
    if kind == 1:
        return rng.integers(-lim, lim, (n, ch))
    x = np.where(np.arange(n)[:, None] % 2 == 0, lim - 1, -lim) * np.where(np.arange(ch) % 2 == 0, 1, -1)[None]
    return np.clip(x, -lim, lim - 1)


@pytest.mark.parametrize('bps', range(16, 33))
def test_every_residue_of_the_length(ctx, bps):
    rng = np.random.default_rng(bps)
    for r in range(4):
        _check(ctx, _content(rng, 1932 + r, 2, bps, 0), 2, bps, 5, 4096)           # one ragged block
        _check(ctx, _content(rng, 40 * (40 + r), 2, bps, 0), 2, bps, 5, 40 + r)    # forty short ones, where neighbouring orders come close
        _check(ctx, _content(rng, 10 * (196 + r), 2, bps, 0), 2, bps, 3, 196 + r)
    _check(ctx, _content(rng, 139, 2, bps, 1), 2, bps, 3, 256)
    _check(ctx, _content(rng, 142, 1, bps, 2), 1, bps, 8, 256)


@pytest.mark.parametrize('shift', [1, 3, 5, 6, 7])
def test_every_residue_with_wasted_bits_of_32(ctx, shift):
    rng = np.random.default_rng(300 + shift)
    for r in range(4):
        for ch in (1, 2):
            _check(ctx, _content(rng, 40 * (40 + r), ch, 32 - shift, 0) << shift, ch, 32, 5, 40 + r)


@pytest.mark.parametrize('bps', [17, 24, 27, 28, 31, 32])
def test_every_residue_of_the_length_generic_kernel(hctx, monkeypatch, bps):
    monkeypatch.setenv('FLACGPU_NO_FAST', '1')
    rng = np.random.default_rng(100 + bps)
    for r in range(4):
        for kind in range(3):
            _check(hctx, _content(rng, 520 + r, 2, bps, kind), 2, bps, 3, 1024)
            _check(hctx, _content(rng, 5 + r, 2, bps, kind), 2, bps, 3, 16)


@pytest.mark.parametrize('ch,bps', [(1, 24), (3, 24), (6, 20), (8, 24), (8, 32)])
def test_other_channel_counts(ctx, ch, bps):
    rng = np.random.default_rng(200 + ch)
    for r in range(4):
        _check(ctx, _content(rng, 300 + r, ch, bps, 0), ch, bps, 4, 4096)


@pytest.mark.parametrize('seed', sorted(cases.UNPINNED_FUZZ_SEEDS))
def test_unpinned_seeds_equal_the_oracle(ctx, seed):
    c = fuzzgen.case(seed)
    _check(ctx, c['pcm'], c['ch'], c['bps'], c['level'], c['bs'], c['sr'], c['subset'], c['limit_min_bitrate'])


@pytest.mark.parametrize('seed', [s for c in CHUNKS for s in range(c * 40, c * 40 + 40)])
def test_seed_bytes_match_the_recorded_ones(ctx, fuzz_golden, seed):
    from pyflac_amd import batch
    if seed in cases.UNPINNED_FUZZ_SEEDS:
        pytest.skip(cases.UNPINNED_REASON)
    g, c = fuzz_golden[str(seed)], fuzzgen.case(seed)
    if g['init_status']:
        with pytest.raises(batch.FlacGpuError):
            batch.settings(c['level'], c['ch'], c['bps'], c['sr'], c['bs'], c['subset'])
        return
    stream = _check(ctx, c['pcm'], c['ch'], c['bps'], c['level'], c['bs'], c['sr'], c['subset'], c['limit_min_bitrate'])
    assert len(stream) == g['total_bytes'] and hashlib.sha256(stream).hexdigest() == g['sha256']
