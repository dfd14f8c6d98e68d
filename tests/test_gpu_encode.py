"""GPU parity tests of the encoder, through the C ABI (batch entry point and FLAC__stream_encoder_*).

Bar: byte-identical to libFLAC 1.4.3 -- checked against the committed golden vectors (SHA-256 of the whole
stream, produced by the reference's binary) and against the CPU oracle frame by frame.
"""
import ctypes as C
import hashlib
import os

import numpy as np
import pytest

from tests import cases

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def ctx():
    import torch
    from pyflac_amd import batch
    assert torch.cuda.is_available()
    return batch.Context(0)


@pytest.fixture(scope='module')
def hctx():
    """A context in the test-hooks build of the library (csrc/Makefile libflacgpu_testhooks.so): the only build that reads the kernel
    selectors (FLACGPU_NO_FAST, FLACGPU_MC, ...) from the environment -- the cross-checks of two implementations of one result."""
    from pyflac_amd import batch
    return batch.Context(0, testhooks=True)


def _gpu_stream(ctx, arr, sr, bps, level, bs, subset, i16=False):
    import torch
    from pyflac_amd import batch
    from pyflac_amd.encoder import stream_header_bytes
    a = np.asarray(arr)
    ch = 1 if a.ndim == 1 else a.shape[1]
    s = batch.settings(level, ch, bps, sr, bs, subset)
    t = torch.from_numpy(np.ascontiguousarray(a.reshape(-1, ch)).astype(np.int16 if i16 else np.int32)).cuda()
    out, offs, st = ctx.encode(s, t)
    body = out[:st.total_bytes].cpu().numpy().tobytes()
    return stream_header_bytes(s) + body, offs.cpu().numpy(), s


@pytest.mark.parametrize('name', sorted(cases.ENCODE_CASES))
def test_batch_encode_matches_golden(ctx, golden, name):
    spec, sr, level, bs, subset = cases.ENCODE_CASES[name]
    g = golden[name]
    pcm, bps = cases.make_pcm(spec)
    stream, offs, _s = _gpu_stream(ctx, cases.as_int_array(pcm, bps), sr, bps, level, bs, subset)
    assert len(stream) == g['total_bytes']
    assert hashlib.sha256(stream).hexdigest() == g['sha256']
    assert [int(x) for x in np.diff(offs)] == [c[0] for c in g['callbacks'][3:]]


@pytest.mark.parametrize('chunk', range(6))
def test_fuzz_corpus_matches_reference_hashes(ctx, fuzz_golden, chunk):
    """Seeded random corpus (tests/fuzzgen.py; hashes recorded from the reference binary): the batch encoder is
    byte-identical and the decoder returns the input, for 1-8 channels, 8-32 bit (32-bit stereo = 33-bit side channel),
    every level, odd block sizes, ragged tails, limit_min_bitrate and non-subset settings."""
    import torch
    from pyflac_amd import batch
    from pyflac_amd.encoder import stream_header_bytes
    from tests import fuzzgen
    for seed in range(chunk * 40, chunk * 40 + 40):
        g = fuzz_golden[str(seed)]
        c = fuzzgen.case(seed)
        if g['init_status']:
            with pytest.raises(batch.FlacGpuError):
                batch.settings(c['level'], c['ch'], c['bps'], c['sr'], c['bs'], c['subset'])
            continue
        s = batch.settings(c['level'], c['ch'], c['bps'], c['sr'], c['bs'], c['subset'])
        s.limit_min_bitrate = 1 if c['limit_min_bitrate'] else 0
        t = torch.from_numpy(np.ascontiguousarray(c['pcm'].astype(np.int32))).cuda()
        out, offs, st = ctx.encode(s, t)
        stream = stream_header_bytes(s) + out[:st.total_bytes].cpu().numpy().tobytes()
        assert len(stream) == g['total_bytes'] and hashlib.sha256(stream).hexdigest() == g['sha256'], seed
        dec, status, _ = ctx.decode(out[:st.total_bytes], offs, c['ch'], c['bps'], len(c['pcm']))
        assert int(status[:, 0].max()) == 0 and torch.equal(dec.reshape(-1, c['ch']), t), seed


@pytest.mark.parametrize('name', sorted(cases.LIMIT_CASES))
def test_limit_min_bitrate_matches_golden(ctx, limit_golden, name):
    """limit_min_bitrate through the batch entry point: byte-identical to the reference binary."""
    import torch
    from pyflac_amd import batch
    from pyflac_amd.encoder import stream_header_bytes
    spec, sr, level, bs = cases.LIMIT_CASES[name]
    pcm, bps = cases.make_pcm(spec)
    arr = cases.as_int_array(pcm, bps)
    s = batch.settings(level, arr.shape[1], bps, sr, bs, True)
    s.limit_min_bitrate = 1
    out, offs, st = ctx.encode(s, torch.from_numpy(np.ascontiguousarray(arr).astype(np.int32)).cuda())
    stream = stream_header_bytes(s) + out[:st.total_bytes].cpu().numpy().tobytes()
    assert [int(x) for x in np.diff(offs.cpu().numpy())] == limit_golden[name]['frame_bytes']
    assert hashlib.sha256(stream).hexdigest() == limit_golden[name]['sha256']


def test_limit_min_bitrate_generic_kernel(hctx, limit_golden, monkeypatch):
    ctx = hctx
    import torch
    from pyflac_amd import batch
    from pyflac_amd.encoder import stream_header_bytes
    monkeypatch.setenv('FLACGPU_NO_FAST', '1')
    for name in ('lmb_equal_st_l5', 'lmb_equal_st_l1', 'lmb_zeros_mono_l5', 'lmb_mixed_st_l8'):
        spec, sr, level, bs = cases.LIMIT_CASES[name]
        pcm, bps = cases.make_pcm(spec)
        arr = cases.as_int_array(pcm, bps)
        s = batch.settings(level, arr.shape[1], bps, sr, bs, True)
        s.limit_min_bitrate = 1
        out, offs, st = ctx.encode(s, torch.from_numpy(np.ascontiguousarray(arr).astype(np.int32)).cuda())
        stream = stream_header_bytes(s) + out[:st.total_bytes].cpu().numpy().tobytes()
        assert hashlib.sha256(stream).hexdigest() == limit_golden[name]['sha256'], name


def test_int16_ingest_equals_int32(ctx):
    pcm, bps = cases.make_pcm({'kind': 'cfg2', 'seconds': 1.0, 'seed': 5})
    a, _, _ = _gpu_stream(ctx, pcm, 48000, 16, 5, 4096, True, i16=False)
    b, _, _ = _gpu_stream(ctx, pcm, 48000, 16, 5, 4096, True, i16=True)
    assert a == b


def test_generic_kernel_equals_fast_kernel(ctx, hctx, monkeypatch):
    """FLACGPU_NO_FAST (test-hooks build) routes every block through the generic kernel; bytes must not change -- and the release
    library does not listen to the variable."""
    from pyflac_amd import _lib
    pcm, bps = cases.make_pcm({'kind': 'hard16', 'seconds': 1.0})
    a, _, _ = _gpu_stream(ctx, pcm, 48000, 16, 8, 4096, True)
    monkeypatch.setenv('FLACGPU_NO_FAST', '1')
    b, _, _ = _gpu_stream(hctx, pcm, 48000, 16, 8, 4096, True)
    assert a == b
    L = _lib.lib()
    buf = (C.c_uint8 * (32 * 64))()
    L.flacgpu_copy_block_results.argtypes = [C.c_void_p, C.c_void_p, C.c_uint32]
    for cx, generic in ((hctx, True), (ctx, False)):
        _gpu_stream(cx, pcm, 48000, 16, 8, 4096, True)
        assert cx._L.flacgpu_copy_block_results(cx._h, buf, 1) == 0
        reserved = np.frombuffer(bytes(buf), np.uint32)[7]            # FgBlockResult.reserved: 4 = a block of the pipeline
        assert (reserved != 4) == generic


def test_many_streams_one_launch(ctx):
    """Config 5 shape: independent streams in one launch equal the same streams encoded one by one."""
    import torch
    from pyflac_amd import batch, synth
    from oracle import oracle as O
    streams = [synth.config5_stream(s, 0.4 + 0.05 * s) for s in range(6)]
    s = batch.settings(5, 2, 16, 48000, 4096, True)
    t = torch.from_numpy(np.concatenate(streams).astype(np.int32)).cuda()
    out, offs, st = ctx.encode(s, t, stream_lengths=[len(x) for x in streams])
    body = out[:st.total_bytes].cpu().numpy().tobytes()
    offs = offs.cpu().numpy()
    cfg, _ = O.config(5, 2, 16, 48000, 4096, True)
    pos = 0
    fi = 0
    for x in streams:
        want, sizes = O.encode_stream(cfg, x)
        nfr = len(sizes)
        got = body[int(offs[fi]):int(offs[fi + nfr])]
        assert got == want[86:]
        fi += nfr
        pos += len(got)
    assert pos == len(body)


def test_stage_records_match_oracle(ctx):
    """Stage-level parity: fixed-predictor sums, autocorrelation (bit-exact doubles), LPC order guess, decisions."""
    import torch
    from pyflac_amd import batch
    from oracle import oracle as O
    pcm, bps = cases.make_pcm({'kind': 'cfg2', 'seconds': 0.5, 'seed': 9})
    arr = pcm.astype(np.int32)
    for level in (5, 8):
        s = batch.settings(level, 2, 16, 48000, 4096, True)
        cfg, _ = O.config(level, 2, 16, 48000, 4096, True)
        out, offs, st = ctx.encode(s, torch.from_numpy(arr).cuda(), debug=True)
        nfull = len(arr) // 4096
        recs = ctx.debug_records(0, nfull)
        for b in range(nfull):
            _b, info = O.encode_frame(cfg, arr[b * 4096:(b + 1) * 4096], b, want_info=True)
            for c in range(4):
                oc, gc = info.cand[c], recs[b].cand[c]
                assert list(oc.fixed_tot) == list(gc.fixed_tot) and oc.fixed_guess == gc.fixed_guess
                assert oc.fixed_bits == gc.fixed_bits
                for v in range(oc.n_vectors):
                    assert list(oc.autoc[v][:cfg.max_lpc_order + 1]) == list(gc.autoc[v][:cfg.max_lpc_order + 1]), (level, b, c, v)
                    assert oc.lpc_guess[v] == gc.lpc_guess[v] and oc.lpc_bits[v] == gc.lpc_bits[v]
                assert (oc.type, oc.order, oc.precision, oc.shift, oc.porder, oc.rice_method, oc.bits) == \
                       (gc.type, gc.order, gc.precision, gc.shift, gc.porder, gc.rice_method, gc.bits)
                assert list(oc.qlp) == list(gc.qlp) and list(oc.rice_params) == list(gc.rice_params)


def test_custom_max_lpc_order_32(ctx):
    """Settings outside the presets (order 32, lax) run on the generic kernel and still match the oracle."""
    import torch
    from pyflac_amd import batch
    from oracle import oracle as O
    pcm, bps = cases.make_pcm({'kind': 'sines', 'bps': 16, 'n': 9000, 'ch': 2, 'level': 0.3})
    arr = pcm.astype(np.int32)
    cfg, _ = O.config(8, 2, 16, 96000, 4096, False)
    cfg.max_lpc_order = 32
    s = batch.settings(8, 2, 16, 96000, 4096, False)
    s.max_lpc_order = 32
    want, sizes = O.encode_stream(cfg, arr)
    out, offs, st = ctx.encode(s, torch.from_numpy(arr).cuda())
    assert out[:st.total_bytes].cpu().numpy().tobytes() == want[86:]
    # and the decoder's generic fallback (predictor order > 12) restores the input
    dec, status, dst = ctx.decode(out[:st.total_bytes], offs.cpu().numpy(), 2, 16, len(arr))
    assert status[:, 0].max() == 0 and np.array_equal(dec.cpu().numpy(), arr)


def test_out_of_range_sample_is_flagged(ctx):
    import torch
    from pyflac_amd import batch
    s = batch.settings(5, 1, 16, 44100, 4096, True)
    bad = np.zeros((4096, 1), np.int32)
    bad[100] = 40000
    with pytest.raises(batch.FlacGpuError):
        ctx.encode(s, torch.from_numpy(bad).cuda())


@pytest.mark.parametrize('seconds,level,kind', [(600.0, 5, 'cfg2'), (300.0, 8, 'cfg4')])
def test_full_size_whole_stream_equals_oracle(ctx, seconds, level, kind):
    """BASELINE sizes (configs[1]: 600 s of 16-bit stereo at level 5; configs[3]: 300 s of 24-bit 96 kHz stereo at level 8), checked
    in full: the GPU stream is the oracle's stream byte for byte (SHA-256 over all 7032 frames: a round trip alone would also pass
    a wrong but decodable choice), the decoder restores the input exactly from the bytes alone, every CRC-16 verifies, the frame
    sizes sum to the stream size."""
    import hashlib
    import torch
    from pyflac_amd import batch
    from oracle import oracle as O
    spec = {'kind': kind, 'seconds': seconds}
    pcm, bps = cases.make_pcm(spec)
    sr = 48000 if kind == 'cfg2' else 96000
    arr = pcm.astype(np.int32)
    s = batch.settings(level, 2, bps, sr, 4096, True)
    t = torch.from_numpy(arr).cuda()
    out, offs, st = ctx.encode(s, t)
    offs_h = offs.cpu().numpy()
    assert st.nblocks == 7032
    assert int(offs_h[-1]) == st.total_bytes and np.all(np.diff(offs_h) > 0)
    dec, status, dst = ctx.decode_stream(out[:st.total_bytes], 2, bps, len(arr), nframes=st.nblocks)
    assert int(status[:, 0].max()) == 0
    assert torch.equal(dec, t)
    del dec
    cfg, _ = O.config(level, 2, bps, sr, 4096, True)
    want, sizes = O.encode_stream(cfg, arr)
    body = out[:st.total_bytes].cpu().numpy().tobytes()
    assert len(sizes) == st.nblocks and np.array_equal(np.diff(offs_h).astype(np.int64), np.asarray(sizes, np.int64))
    assert hashlib.sha256(body).hexdigest() == hashlib.sha256(want[86:]).hexdigest()


def test_batch_stream_whole_equals_oracle(ctx):
    """configs[4] shape at its real stream length: four 60 s streams in one launch; the FIRST AND THE LAST stream whole equal the
    oracle's streams (SHA-256), and all four decode back from the bytes alone."""
    import hashlib
    import torch
    from pyflac_amd import batch, synth
    from oracle import oracle as O
    streams = [synth.config5_stream(s, 60.0) for s in range(4)]
    s = batch.settings(5, 2, 16, 48000, 4096, True)
    t = torch.from_numpy(np.concatenate(streams).astype(np.int32)).cuda()
    out, offs, st = ctx.encode(s, t, stream_lengths=[len(x) for x in streams])
    h = offs.cpu().numpy().astype(np.int64)
    nfr = -(-len(streams[0]) // 4096)
    cfg, _ = O.config(5, 2, 16, 48000, 4096, True)
    for k in (0, 3):
        want, sizes = O.encode_stream(cfg, streams[k].astype(np.int32))
        got = out[int(h[k * nfr]):int(h[(k + 1) * nfr])].cpu().numpy().tobytes()
        assert len(sizes) == nfr and hashlib.sha256(got).hexdigest() == hashlib.sha256(want[86:]).hexdigest()
    ranges = [(int(h[(k + 1) * nfr] - h[k * nfr]), nfr) for k in range(4)]
    dec, status, dst = ctx.decode_streams(out[:st.total_bytes], ranges, 2, 16, t.shape[0])
    assert int(status[:, 0].max()) == 0 and torch.equal(dec, t)


def test_batch_128_streams_whole(ctx):
    """configs[4] at its per-GPU size: 128 independent 60 s streams (90 112 blocks: tiled scans, the decoder's frame index over all
    streams) in ONE launch.  The first, the middle and the last stream whole equal the oracle's streams (SHA-256), and everything
    decodes back from the bytes alone (one decode launch over all streams)."""
    import hashlib
    import torch
    from pyflac_amd import batch, synth
    from oracle import oracle as O
    nstreams = 128
    streams = [synth.config5_stream(s, 60.0) for s in range(nstreams)]
    s = batch.settings(5, 2, 16, 48000, 4096, True)
    t = torch.from_numpy(np.concatenate(streams).astype(np.int32)).cuda()
    out, offs, st = ctx.encode(s, t, stream_lengths=[len(x) for x in streams])
    h = offs.cpu().numpy().astype(np.int64)
    nfr = -(-len(streams[0]) // 4096)
    assert st.nblocks == nstreams * nfr == 90112
    cfg, _ = O.config(5, 2, 16, 48000, 4096, True)
    for k in (0, nstreams // 2, nstreams - 1):
        want, sizes = O.encode_stream(cfg, streams[k].astype(np.int32))
        got = out[int(h[k * nfr]):int(h[(k + 1) * nfr])].cpu().numpy().tobytes()
        assert len(sizes) == nfr and hashlib.sha256(got).hexdigest() == hashlib.sha256(want[86:]).hexdigest(), k
    ranges = [(int(h[(k + 1) * nfr] - h[k * nfr]), nfr) for k in range(nstreams)]
    dec, status, dst = ctx.decode_streams(out[:st.total_bytes], ranges, 2, 16, t.shape[0])
    assert int(status[:, 0].max()) == 0 and torch.equal(dec, t)


# ---------------------------------------------------------------------------------------------- round-2 additions
def test_log_guard_forced_keeps_bytes_and_counts(golden):
    """Near-tie guard of the LPC order guess (flacgpu_set_log_guard): with the threshold forced above every margin all order
    guesses are repeated with the correctly rounded double-double logarithm -- the bytes must not change (the two logs agree
    wherever the margin is comfortable) and the counter must move.  With the default threshold the counter stays at zero
    exactly when the smallest margin seen is above it."""
    import torch
    from pyflac_amd import batch, _lib
    c2 = batch.Context(0)
    L = _lib.lib()
    for name in ('cfg2_20s_l5', 'cfg4_10s_l8', 'noise16_st', 'sines24_l8_bs4608'):
        spec, sr, level, bs, subset = cases.ENCODE_CASES[name]
        pcm, bps = cases.make_pcm(spec)
        L.flacgpu_set_log_guard(c2._h, 1e30)
        stream, _offs, _s = _gpu_stream(c2, cases.as_int_array(pcm, bps), sr, bps, level, bs, subset)
        assert hashlib.sha256(stream).hexdigest() == golden[name]['sha256'], name
        a = np.asarray(cases.as_int_array(pcm, bps))
        s = batch.settings(level, a.shape[1], bps, sr, bs, subset)
        t = torch.from_numpy(np.ascontiguousarray(a).astype(np.int32)).cuda()
        _o, _f, st = c2.encode(s, t)
        assert st.log_guard_subframes > 0, name
        assert 0.0 <= st.lpc_order_min_margin < 1e30
        L.flacgpu_set_log_guard(c2._h, 1e-6)
        _o, _f, st = c2.encode(s, t)
        assert (st.log_guard_subframes == 0) == (st.lpc_order_min_margin >= 1e-6), (name, st.log_guard_subframes, st.lpc_order_min_margin)


def test_log_guard_margin_over_fuzz_corpus(ctx, fuzz_golden):
    """Hunt for near-ties: the smallest margin between the two best LPC order estimates over the seeded fuzz corpus (the
    cases the pipeline encodes).  Whenever it falls below the guard threshold the guard must have fired -- the bytes of
    these cases are compared with the reference's in test_fuzz_corpus_matches_reference_hashes."""
    import torch
    from pyflac_amd import batch
    from tests import fuzzgen
    smallest, seen = float('inf'), 0
    for seed in range(240):
        g = fuzz_golden[str(seed)]
        c = fuzzgen.case(seed)
        if g['init_status'] or c['level'] < 3 or c['ch'] > 2 or c['bps'] > 24:
            continue
        s = batch.settings(c['level'], c['ch'], c['bps'], c['sr'], c['bs'], c['subset'])
        t = torch.from_numpy(np.ascontiguousarray(c['pcm'].astype(np.int32))).cuda()
        _o, _f, st = ctx.encode(s, t)
        if st.lpc_order_min_margin < 1e29:
            seen += 1
            smallest = min(smallest, st.lpc_order_min_margin)
            assert (st.log_guard_subframes > 0) == (st.lpc_order_min_margin < 1e-6), seed
    assert seen > 20
    print('smallest LPC order margin over %d fuzz cases: %.3e bits' % (seen, smallest))


def test_window_selfcheck(golden, monkeypatch):
    """The tukey tapers of the preset shapes at block size 4096 are committed; a host whose cosf disagrees gets the committed
    values and a note.  FLACGPU_WINDOW_SELFTEST corrupts the generated table first: the bytes must still be the golden ones."""
    from pyflac_amd import batch, _lib
    L = _lib.lib()
    c1 = batch.Context(0)
    for name in ('cfg2_20s_l5', 'cfg4_10s_l8'):
        spec, sr, level, bs, subset = cases.ENCODE_CASES[name]
        pcm, bps = cases.make_pcm(spec)
        stream, _o, _s = _gpu_stream(c1, cases.as_int_array(pcm, bps), sr, bps, level, bs, subset)
        assert hashlib.sha256(stream).hexdigest() == golden[name]['sha256']
    assert L.flacgpu_window_note(c1._h) == b'', 'this host\'s cosf disagrees with the committed window table'
    monkeypatch.setenv('FLACGPU_WINDOW_SELFTEST', '1')
    c3 = batch.Context(0)                    # (the release library does not listen to the hook)
    stream, _o, _s = _gpu_stream(c3, cases.as_int_array(*cases.make_pcm(cases.ENCODE_CASES['cfg2_20s_l5'][0])), 48000, 16, 5, 4096, True)
    assert L.flacgpu_window_note(c3._h) == b''
    c2 = batch.Context(0, testhooks=True)
    L = c2._L
    for name in ('cfg2_20s_l5', 'cfg4_10s_l8'):
        spec, sr, level, bs, subset = cases.ENCODE_CASES[name]
        pcm, bps = cases.make_pcm(spec)
        stream, _o, _s = _gpu_stream(c2, cases.as_int_array(pcm, bps), sr, bps, level, bs, subset)
        assert hashlib.sha256(stream).hexdigest() == golden[name]['sha256']
    assert b'committed table is used' in L.flacgpu_window_note(c2._h)


def test_frames_of_24_bit_input_are_packed_at_their_final_place(ctx, hctx, monkeypatch):
    """Round 6: 17..24-bit input takes the direct packing kernel too (its 64-bit forms), and so does 32-bit
    input in blocks of up to 4096 samples: direct_path == 1, no block handed back, bytes and offsets the oracle's -- and the chunk
    form (FLACGPU_DIRECT24=0, test-hooks library) gives the same."""
    import torch
    from pyflac_amd import batch, synth
    from oracle import oracle as O
    rng = np.random.default_rng(24)
    for level, ch, bps, bs, n, noise in ((8, 2, 24, 4096, 4096 * 6 + 300, False), (5, 1, 24, 4096, 4096 * 3 + 17, False), (5, 2, 20, 4608, 4608 * 3 + 100, False),
                                         (8, 2, 24, 1152, 1152 * 7, False), (3, 2, 24, 4096, 4096 * 3, True), (0, 2, 24, 2304, 2304 * 3 + 5, False),
                                         (5, 2, 32, 4096, 4096 * 3 + 9, False), (8, 2, 32, 4096, 4096 * 2, True), (5, 1, 32, 1024, 1024 * 5, True)):
        pcm = synth.config4_stereo24(n / 48000.0 + 0.01, bs + ch)[:n].astype(np.int32)
        pcm = pcm >> (24 - bps) if bps <= 24 else pcm * 251 + rng.integers(-90, 90, pcm.shape).astype(np.int32)      # (32 bit: no wasted bits)
        if noise:
            pcm = rng.integers(-2**(bps - 1), 2**(bps - 1), pcm.shape).astype(np.int32)     # verbatim subframes: the largest frames there are
        pcm = np.ascontiguousarray(pcm[:, :ch])
        s = batch.settings(level, ch, bps, 48000, bs, True)
        cfg, _ = O.config(level, ch, bps, 48000, bs, True)
        want, sizes = O.encode_stream(cfg, pcm)
        dev = torch.from_numpy(pcm).cuda()
        for c, direct in ((ctx, 1), (hctx, 0)):
            if not direct:
                monkeypatch.setenv('FLACGPU_DIRECT24', '0')
            out, offs, st = c.encode(s, dev)
            monkeypatch.delenv('FLACGPU_DIRECT24', raising=False)
            assert st.direct_path == direct and st.redo_blocks == 0, (level, ch, bps, bs, st.direct_path, st.redo_blocks)
            body = out[:st.total_bytes].cpu().numpy().tobytes()
            assert body == want[len(want) - int(sizes.sum()):], (level, ch, bps, bs, direct)
            assert np.array_equal(np.diff(offs.cpu().numpy().astype(np.int64)), sizes.astype(np.int64))


def test_the_autocorrelation_of_a_few_blocks_by_a_workgroup_each_equals_the_wave_a_block_form(ctx, hctx, monkeypatch):
    """Round 6: launches of up to 256 blocks -- StreamEncoder.process() above all -- take fg_pipe_autoc1_kernel (a workgroup a block: one
    wave on the chains of matrix instructions, eight that stage the chunks ahead of it); larger ones keep fg_pipe_autoc_kernel (a wave
    a block).  Same sums in the same order: the bytes are the oracle's either way -- every level's windows (partial and punched ones
    at level 8), one and two channels, 16 / 24 / 32 bit, int16 input, odd block sizes and tails, a single short block -- with the
    release library's choice (at levels 6 - 8 and up to 42 blocks: the windows that run a chain side by side, a workgroup each, and
    fg_pipe_autoc_fix_kernel behind them), with the old kernel forced on the small launch (FLACGPU_AUTOC1=0), the new one on every
    launch (2) and with its windows one behind the other (3) -- test-hooks library."""
    import torch
    from pyflac_amd import batch, synth
    from oracle import oracle as O
    rng = np.random.default_rng(61)
    cases = [(5, 2, 16, 4096, 4096 * 5 + 1234, False), (8, 2, 24, 4096, 4096 * 3 + 77, False), (8, 2, 16, 1152, 1152 * 6 + 5, True), (0, 1, 16, 4096, 4096 * 2 + 9, False),
             (3, 2, 16, 4095, 4095 * 3, False), (8, 1, 24, 2304, 2304 * 2 + 130, False), (5, 2, 32, 4096, 4096 * 2 + 300, False), (8, 2, 16, 4608, 4608 + 64, False),
             (6, 2, 16, 4096, 100, False), (7, 2, 24, 576, 576 * 9, False), (8, 2, 16, 1024, 1024 * 50 + 3, False), (6, 1, 16, 4096, 4096 * 4, False)]
    for level, ch, bps, bs, n, i16 in cases:
        base = synth.config2_stereo16(n / 48000.0 + 0.01, level + bs)[:n].astype(np.int64)
        if bps == 24:
            base = base * 211 + rng.integers(-60, 60, base.shape)
        if bps == 32:
            base = base * 52001 + rng.integers(-9000, 9000, base.shape)
        pcm = np.ascontiguousarray(base[:, :ch].astype(np.int32))
        s = batch.settings(level, ch, bps, 48000, bs, bs != 4095)
        cfg, _ = O.config(level, ch, bps, 48000, bs, bs != 4095)
        want, sizes = O.encode_stream(cfg, pcm)
        dev = torch.from_numpy(pcm.astype(np.int16) if i16 else pcm).cuda()
        for c, sel in ((ctx, None), (hctx, '0'), (hctx, '2'), (hctx, '3')):
            if sel is not None:
                monkeypatch.setenv('FLACGPU_AUTOC1', sel)
            out, offs, st = c.encode(s, dev)
            monkeypatch.delenv('FLACGPU_AUTOC1', raising=False)
            body = out[:st.total_bytes].cpu().numpy().tobytes()
            assert body == want[len(want) - int(sizes.sum()):], (level, ch, bps, bs, n, sel)
    # a launch beyond the limit, both ways (300 blocks)
    pcm = synth.config2_stereo16(300 * 4096 / 48000.0 + 0.01, 3)[:300 * 4096].astype(np.int32)
    s = batch.settings(5, 2, 16, 48000, 4096, True)
    dev = torch.from_numpy(pcm).cuda()
    outs = []
    for sel in (None, '2'):
        if sel is not None:
            monkeypatch.setenv('FLACGPU_AUTOC1', sel)
        out, offs, st = hctx.encode(s, dev)
        monkeypatch.delenv('FLACGPU_AUTOC1', raising=False)
        outs.append(out[:st.total_bytes].cpu().numpy().tobytes())
    cfg, _ = O.config(5, 2, 16, 48000, 4096, True)
    want, sizes = O.encode_stream(cfg, pcm)
    assert outs[0] == outs[1] == want[len(want) - int(sizes.sum()):]


def test_wasted_bits_stay_in_the_pipeline(ctx):
    """Blocks whose samples share trailing zero bits (16-bit audio in a 24-bit container) are encoded by the pipeline itself
    (no hand-over to the generic kernel) and equal the oracle's bytes."""
    import torch
    from pyflac_amd import batch
    from oracle import oracle as O
    rng = np.random.default_rng(5)
    n = 4096 * 6
    t_ = np.arange(n)
    base = (8000 * np.sin(t_ * 0.01) + rng.integers(-300, 300, n)).astype(np.int64)
    a = np.stack([base << 8, (base // 2 + 5) << 8], axis=1).astype(np.int32)     # 24-bit samples, 8 wasted bits
    for level in (5, 8):
        s = batch.settings(level, 2, 24, 96000, 4096, True)
        cfg, _ = O.config(level, 2, 24, 96000, 4096, True)
        out, offs, st = ctx.encode(s, torch.from_numpy(a).cuda())
        assert st.redo_blocks == 0
        want, _res = O.encode_stream(cfg, a)
        body = out[:st.total_bytes].cpu().numpy().tobytes()
        assert want.endswith(body) and len(body) > 0


def test_timing_levels_and_repeated_layouts(ctx):
    """flacgpu_set_stage_timing: level 0 ends a call through the pinned signal area (GPU time from the wall-clock stamps, no
    event fields), level 1 fills the HIP-event fields, level 2 also the stage times -- the bytes are the same at every
    level.  And the block list kept from the previous call (same settings, same stream list) is dropped when anything
    about the call changes: A, B, A again gives A's bytes again, for a different level, a different split into streams
    and a different length."""
    import torch
    from pyflac_amd import _lib, batch, synth
    L = _lib.lib()
    pcm = torch.from_numpy(synth.config2_stereo16(6.0, 3).astype(np.int32)).cuda()
    s5 = batch.settings(5, 2, 16, 48000, 4096, True)
    s8 = batch.settings(8, 2, 16, 48000, 4096, True)

    def enc(s, t, lengths=None):
        out, offs, st = ctx.encode(s, t, stream_lengths=lengths)
        return out[:st.total_bytes].cpu().numpy().tobytes(), offs.cpu().numpy().copy(), st

    try:
        ref, roffs, st0 = enc(s5, pcm)
        assert st0.total_gpu_ms > 0 and st0.encode_kernel_ms == 0 and sum(st0.stage_ms) == 0
        for level in (1, 2):
            L.flacgpu_set_stage_timing(ctx._h, level)
            b, o, st = enc(s5, pcm)
            assert b == ref and np.array_equal(o, roffs)
            assert st.total_gpu_ms > 0 and st.encode_kernel_ms > 0 and st.total_gpu_ms >= st.encode_kernel_ms
            assert (sum(st.stage_ms) > 0) == (level == 2)
            dec, status, dst = ctx.decode_stream(torch.from_numpy(np.frombuffer(b, np.uint8).copy()).cuda(), 2, 16, pcm.shape[0], nframes=st.nblocks)
            assert torch.equal(dec[:pcm.shape[0]], pcm) and dst.total_gpu_ms > 0 and dst.decode_kernel_ms > 0
        # level 3: the default call between two events -- same bytes, the total from the events, no break-down
        L.flacgpu_set_stage_timing(ctx._h, 3)
        b, o, st = enc(s5, pcm)
        assert b == ref and np.array_equal(o, roffs)
        assert st.total_gpu_ms > 0 and st.encode_kernel_ms == 0 and sum(st.stage_ms) == 0
        dec, status, dst = ctx.decode_stream(torch.from_numpy(np.frombuffer(b, np.uint8).copy()).cuda(), 2, 16, pcm.shape[0], nframes=st.nblocks)
        assert torch.equal(dec[:pcm.shape[0]], pcm) and dst.total_gpu_ms > 0 and dst.decode_kernel_ms == 0
    finally:
        L.flacgpu_set_stage_timing(ctx._h, 0)
    other8, _o, _s = enc(s8, pcm)
    assert other8 != ref
    assert enc(s5, pcm)[0] == ref
    half = pcm.shape[0] // 2
    two, o2, st2 = enc(s5, pcm, [half, pcm.shape[0] - half])
    assert st2.nblocks == -(-half // 4096) + -(-(pcm.shape[0] - half) // 4096) and two != ref
    assert enc(s5, pcm)[0] == ref
    short, _o, _s = enc(s5, pcm[:half].contiguous())
    assert short != ref and enc(s5, pcm)[0] == ref
    assert enc(s5, pcm[:half].contiguous())[0] == short


def test_wasted_bits_differ_between_candidates(ctx):
    """The unary wasted-bits field belongs to every subframe estimate (libFLAC adds subframe->wasted_bits): when the four
    candidates of a stereo block have different wasted bits it decides the channel assignment.  A DC signal with an odd left
    and a right channel that is a multiple of four (fuzz seed 33402, found in round 2: the pipeline chose mid/side where
    libFLAC keeps the channels independent), and a music-like signal whose left channel has its two low bits cleared --
    bytes against the oracle at the levels that try mid/side, stage records at level 5."""
    import torch
    from pyflac_amd import batch
    from pyflac_amd.encoder import stream_header_bytes
    from oracle import oracle as O
    dc = np.empty((8310, 2), np.int32)
    dc[:, 0], dc[:, 1] = 23693, 25684
    pcm, _bps = cases.make_pcm({'kind': 'cfg2', 'seconds': 0.4, 'seed': 21})
    mus = pcm.astype(np.int32).copy()
    mus[:, 0] &= ~3
    for name, arr, bs in (('dc', dc, 2048), ('low bits cleared', mus, 4096)):
        for level in (1, 2, 4, 5, 7, 8):
            s = batch.settings(level, 2, 16, 44100, bs, True)
            cfg, _ = O.config(level, 2, 16, 44100, bs, True)
            want, _ = O.encode_stream(cfg, arr)
            out, offs, st = ctx.encode(s, torch.from_numpy(arr).cuda())
            got = stream_header_bytes(s) + out[:st.total_bytes].cpu().numpy().tobytes()
            assert got == want, (name, level)
    s = batch.settings(5, 2, 16, 44100, 4096, True)
    cfg, _ = O.config(5, 2, 16, 44100, 4096, True)
    ctx.encode(s, torch.from_numpy(mus).cuda(), debug=True)
    nfull = len(mus) // 4096
    recs = ctx.debug_records(0, nfull)
    seen = set()
    for b in range(nfull):
        _b, info = O.encode_frame(cfg, mus[b * 4096:(b + 1) * 4096], b, want_info=True)
        for c in range(4):
            oc, gc = info.cand[c], recs[b].cand[c]
            seen.add(int(oc.wasted))
            assert (oc.wasted, oc.sbps, oc.type, oc.order, oc.bits, oc.fixed_bits) == (gc.wasted, gc.sbps, gc.type, gc.order, gc.bits, gc.fixed_bits), (b, c)
            for v in range(oc.n_vectors):
                assert oc.lpc_bits[v] == gc.lpc_bits[v], (b, c, v)
    assert len(seen) > 1


@pytest.mark.parametrize('seed', [79464, 93095])
def test_loose_mid_side_decision_frame_with_limit_min_bitrate(ctx, seed):
    """Fuzz seeds 79464 / 93095 (found in round 2): levels 1 and 4 decide between independent and mid/side coding on every
    n-th frame and copy the decision in between.  libFLAC evaluates all four candidates on a DECISION frame, so
    limit_min_bitrate (no frame of CONSTANT subframes only) applies to its mid and side channels as in any full frame; the
    frames that merely copy the decision evaluate mid/side alone and are never limited.  The decision frame used to be
    encoded like a copying one: a silent first block came out with a CONSTANT mid channel."""
    import torch
    from pyflac_amd import batch
    from pyflac_amd.encoder import stream_header_bytes
    from oracle import oracle as O
    from tests import fuzzgen
    c = fuzzgen.case(seed)
    assert c['limit_min_bitrate'] and c['level'] in (1, 4)
    cfg, _rc = O.config(c['level'], c['ch'], c['bps'], c['sr'], c['bs'], c['subset'])
    s = batch.settings(c['level'], c['ch'], c['bps'], c['sr'], c['bs'], c['subset'])
    cfg.limit_min_bitrate = 1
    s.limit_min_bitrate = 1
    a32 = np.ascontiguousarray(c['pcm'].astype(np.int32))
    want, _ = O.encode_stream(cfg, a32)
    out, offs, st = ctx.encode(s, torch.from_numpy(a32).cuda())
    assert stream_header_bytes(s) + out[:st.total_bytes].cpu().numpy().tobytes() == want


def _multichannel_pcm(seed, channels, n, bps):
    rng = np.random.default_rng(seed)
    t = np.arange(n)
    amp = (1 << (bps - 2)) * 0.5
    cols = []
    for c in range(channels):
        x = amp * np.sin(0.003 * (c + 2) * t + c) + rng.normal(0, amp / 40, n)
        if c == channels - 1:
            x = np.full(n, 123.0)                       # a constant channel
        if c == 1:
            x = np.round(x / 16) * 16                   # four wasted bits
        cols.append(np.clip(np.round(x), -(1 << (bps - 1)), (1 << (bps - 1)) - 1))
    return np.stack(cols, axis=1).astype(np.int32)


@pytest.mark.parametrize('channels,bps,level,bs,n', [(3, 16, 5, 4096, 4096 * 5 + 777), (6, 16, 5, 4096, 4096 * 9), (8, 16, 8, 4096, 4096 * 3 + 100),
                                                     (4, 24, 8, 4096, 4096 * 4 + 63), (6, 16, 0, 1152, 1152 * 7 + 1), (5, 8, 3, 576, 576 * 11 + 17)])
def test_more_than_two_channels_through_the_pipeline(ctx, hctx, monkeypatch, channels, bps, level, bs, n):
    """Streams of three to eight channels: every channel a one-channel view through the pipeline, the frames spliced by
    flac_enc_merge.hip (fg_ctx.cpp encode_multichannel).  Bytes equal the oracle's and the generic kernel's (FLACGPU_MC=0),
    frame index included."""
    from oracle import oracle as O
    pcm = _multichannel_pcm(channels * 100 + level, channels, n, bps)
    got, offs, s = _gpu_stream(ctx, pcm, 48000, bps, level, bs, True)
    cfg, _ = O.config(level, channels, bps, 48000, bs, True)
    want, sizes = O.encode_stream(cfg, pcm)
    assert got[86:] == want[86:]
    assert list(np.diff(offs)) == list(sizes)
    monkeypatch.setenv('FLACGPU_MC', '0')
    ref, offs2, _ = _gpu_stream(hctx, pcm, 48000, bps, level, bs, True)
    assert ref == got and np.array_equal(offs, offs2)


def test_more_than_two_channels_many_streams_int16(ctx):
    """Several six-channel streams of different lengths in one launch, 16-bit ingest: stream by stream the oracle's bytes."""
    import torch
    from pyflac_amd import batch
    from oracle import oracle as O
    lens = [4096 * 3 + 5, 4096, 17, 4096 * 2 + 2048]
    streams = [_multichannel_pcm(40 + i, 6, n, 16) for i, n in enumerate(lens)]
    s = batch.settings(5, 6, 16, 48000, 4096, True)
    t = torch.from_numpy(np.concatenate(streams).astype(np.int16)).cuda()
    out, offs, st = ctx.encode(s, t, stream_lengths=lens)
    body = out[:st.total_bytes].cpu().numpy().tobytes()
    offs = offs.cpu().numpy()
    cfg, _ = O.config(5, 6, 16, 48000, 4096, True)
    fi = 0
    for x in streams:
        want, sizes = O.encode_stream(cfg, x)
        assert body[int(offs[fi]):int(offs[fi + len(sizes)])] == want[86:]
        fi += len(sizes)
    assert int(offs[fi]) == len(body) and st.error_flags == 0


def test_large_coefficients_do_not_overflow_the_warm_up(ctx):
    """Fuzz seed 754506 (24-bit square wave, level 8): under a punched subdivide_tukey window the order-9 predictor has
    coefficients near -9005 at shift 0.  Its residual is zero, but the 'residual' of a warm-up sample -- formed over a history
    of zeros, which libFLAC never does -- exceeds 32 bits; the evaluation must not count that as an overflow of the candidate."""
    from oracle import oracle as O
    from tests import fuzzgen
    c = fuzzgen.case(754506)
    assert (c['ch'], c['bps'], c['level'], c['kind']) == (2, 24, 8, 'square')
    import torch
    from pyflac_amd import batch
    s = batch.settings(c['level'], c['ch'], c['bps'], c['sr'], c['bs'], c['subset'])
    s.limit_min_bitrate = 1 if c['limit_min_bitrate'] else 0
    cfg, _ = O.config(c['level'], c['ch'], c['bps'], c['sr'], c['bs'], c['subset'])
    cfg.limit_min_bitrate = s.limit_min_bitrate
    arr = c['pcm'].astype(np.int32).reshape(-1, c['ch'])
    out, offs, st = ctx.encode(s, torch.from_numpy(arr).cuda())
    want, sizes = O.encode_stream(cfg, arr)
    assert out[:st.total_bytes].cpu().numpy().tobytes() == want[86:]


def _in32(pcm24, shift=8):
    return (pcm24.astype(np.int64) << shift).astype(np.int32)


@pytest.mark.parametrize('level', [0, 3, 5, 8])
def test_24_bit_material_in_32_bit_container_stays_in_the_pipeline(ctx, level):
    """pyFLAC encodes an int32 array as a 32-bit stream (pyflac/encoder.py:109), and soundfile hands a 24-bit WAV over as
    left-justified int32: 32-bit FLAC whose samples share eight wasted bits.  The pipeline stages them shifted down (pipe_preshift);
    bytes equal the oracle's, no block goes to the generic kernel."""
    import torch
    from pyflac_amd import batch
    from oracle import oracle as O
    from pyflac_amd import synth
    pcm24 = synth.config4_stereo24(0.7, 3)                 # (BASELINE config 3/4 signal: 24-bit stereo, 96 kHz)
    assert pcm24.shape[1] == 2 and int(np.abs(pcm24).max()) < (1 << 23)
    arr = _in32(pcm24)
    n = (len(arr) // 4096) * 4096 + 333
    arr = np.ascontiguousarray(arr[:n])
    s = batch.settings(level, 2, 32, 96000, 4096, True)
    cfg, _ = O.config(level, 2, 32, 96000, 4096, True)
    out, offs, st = ctx.encode(s, torch.from_numpy(arr).cuda())
    want, sizes = O.encode_stream(cfg, arr)
    assert out[:st.total_bytes].cpu().numpy().tobytes() == want[86:]
    assert st.redo_blocks == 0


def test_32_bit_streams_mixed_content(ctx):
    """A 32-bit stereo stream whose blocks differ: 24-bit material (pipeline), one channel silent, both silent, 16-bit material
    (sixteen shared wasted bits), true 32-bit noise (the pipeline's fp64 forms, round 4), L == R (a zero side channel).  Every frame the
    oracle's; round 6: the ragged tail of true 32-bit content stays in the pipeline too (pipe_eval_cand_w32<..., RAG>)."""
    import torch
    from pyflac_amd import batch
    from oracle import oracle as O
    rng = np.random.default_rng(11)
    bs = 4096
    t = np.arange(bs)
    tone = lambda a, f, ph: np.round(a * np.sin(2 * np.pi * f * t / 48000 + ph) + rng.normal(0, a / 300, bs)).astype(np.int64)
    blocks = []
    b24 = np.stack([tone(3e6, 440, 0), tone(2e6, 660, 1)], axis=1)
    blocks.append(b24 << 8)                                                     # 24-bit material
    blocks.append(np.stack([tone(3e6, 440, 0) << 8, np.zeros(bs, np.int64)], axis=1))    # right channel silent
    blocks.append(np.zeros((bs, 2), np.int64))                                  # digital silence
    blocks.append(np.stack([tone(2e4, 300, 0), tone(1e4, 500, 2)], axis=1) << 16)        # 16-bit material
    blocks.append(rng.integers(-2**31, 2**31, (bs, 2)))                          # true 32-bit content
    x = tone(2.5e6, 880, 0) << 8
    blocks.append(np.stack([x, x], axis=1))                                     # L == R
    blocks.append(np.stack([tone(3e6, 100, 0) << 8, tone(3e6, 150, 0) << 9], axis=1))    # different counts per channel
    blocks.append(rng.integers(-2**31, 2**31, (777, 2)))                         # a true 32-bit tail
    arr = np.concatenate(blocks).astype(np.int32)
    for level in (5, 8):
        s = batch.settings(level, 2, 32, 48000, bs, True)
        cfg, _ = O.config(level, 2, 32, 48000, bs, True)
        out, offs, st = ctx.encode(s, torch.from_numpy(arr).cuda())
        want, sizes = O.encode_stream(cfg, arr)
        assert list(np.diff(offs.cpu().numpy())) == list(sizes)
        assert out[:st.total_bytes].cpu().numpy().tobytes() == want[86:]
        assert st.redo_blocks == 0                       # (round 5: 1 -- the 777-sample tail of true 32-bit content, ragged geometry)


@pytest.mark.parametrize('level', [2, 5, 8])
def test_ragged_blocks_of_true_32_bit_content_stay_in_the_pipeline(ctx, level):
    """Round 6 (the third time asked): tails and odd block sizes of TRUE 32-bit content -- 33-bit side channel, fewer than eight shared
    wasted bits -- are evaluated and packed by the pipeline's fp64 forms in the ragged lane geometry instead of going to the generic
    kernel.  Stereo and mono, tails of many lengths (one sample more in some lanes of a group, idle lanes, short partitions), an odd
    block size, a few wasted bits -- and every residue of (length - 4) mod 4."""
    import torch
    from pyflac_amd import batch
    from oracle import oracle as O
    rng = np.random.default_rng(600 + level)
    for ch, bs, n, shift, redo_want in ((2, 4096, 4096 + 777, 0, 0), (2, 4096, 4096 + 1000, 0, 0), (1, 4096, 4096 + 2049, 0, 0), (2, 1155, 3 * 1155 + 401, 0, 0),
                                        (2, 4096, 4096 + 516, 2, 0), (2, 4096, 4096 + 35, 0, 0), (2, 4096, 4096 + 777, 6, 0), (2, 4096, 4096 + 778, 0, 0),
                                        (2, 4096, 4096 + 779, 0, 0), (1, 4096, 4096 + 778, 6, 0), (2, 4096, 4096 + 779, 5, 0), (2, 256, 66, 0, 0), (2, 64, 107, 0, 0)):
        walk = np.cumsum(rng.integers(-2**26, 2**26, (n, ch)), axis=0)
        x = ((walk + rng.integers(-2**20, 2**20, (n, ch))) % 2**32 - 2**31).astype(np.int64)
        x = (x >> shift) << shift                       # `shift` wasted bits
        arr = np.ascontiguousarray(np.clip(x, -2**31, 2**31 - 1).astype(np.int32))
        s = batch.settings(level, ch, 32, 48000, bs, bs == 4096)
        cfg, _ = O.config(level, ch, 32, 48000, bs, bs == 4096)
        out, offs, st = ctx.encode(s, torch.from_numpy(arr).cuda())
        want, sizes = O.encode_stream(cfg, arr)
        assert list(np.diff(offs.cpu().numpy())) == list(sizes), (ch, bs, n, shift)
        assert out[:st.total_bytes].cpu().numpy().tobytes() == want[len(want) - int(sizes.sum()):], (ch, bs, n, shift)
        if redo_want is not None:
            assert st.redo_blocks == redo_want, (ch, bs, n, shift, st.redo_blocks)


def test_md5_of_device_resident_streams(ctx):
    """flacgpu_md5_streams: STREAMINFO's md5sum for streams the batch entry point encoded (it leaves the field to the caller) --
    equal to MD5 over the samples as libFLAC hashes them, for 8 .. 32 bit, 1 .. 6 channels, int16 and int32 input, lengths around
    the 64-byte block boundaries, and equal to the oracle's md5_pcm."""
    import hashlib
    import torch
    from oracle import oracle as O
    rng = np.random.default_rng(3)
    for ch, bps, dt in [(2, 16, np.int32), (2, 16, np.int16), (1, 8, np.int32), (2, 24, np.int32), (6, 16, np.int16), (2, 32, np.int32), (1, 12, np.int32), (3, 20, np.int32)]:
        lengths = [1, 13, 14, 15, 16, 27, 28, 31, 32, 33, 1000, 4096 * 3 + 5, 7]
        lim = 1 << (bps - 1)
        a = rng.integers(-lim, lim, size=(sum(lengths), ch), dtype=np.int64).astype(dt)
        digs, ms = ctx.md5_streams(torch.from_numpy(a).cuda(), bps, lengths)
        nb = (bps + 7) // 8
        pos = 0
        for n, got in zip(lengths, digs):
            x = a[pos:pos + n].astype(np.int64)
            raw = b''.join(int(v & ((1 << (8 * nb)) - 1)).to_bytes(nb, 'little') for v in x.reshape(-1))
            assert got == hashlib.md5(raw).digest(), (ch, bps, dt, n)
            assert got == O.md5_pcm(a[pos:pos + n].astype(np.int32), bps), (ch, bps, n)
            pos += n


def test_guard_statistics_survive_a_redo_pass(monkeypatch):
    """a call that hands a block back to the generic kernel (FG_ERR_REDO) ends through a SECOND finish pass, whose
    signal kernel finds the near-tie counters already reset by the first one: the statistics of the call (log_guard_subframes,
    lpc_order_min_margin) must be the first pass's -- equal to what the event-timed form of the same call (stage_timing 1, which
    reads the counters without resetting them) reports, and not 0 / +inf.
    (Round 6: no content class leaves the pipeline any more -- true 32-bit tails included --, so the hand-over is provoked: the
    test-hooks library in the chunk form with a frame-bit window of 28 words, FLACGPU_FBW, which a lane of 32 verbatim 32-bit samples
    does not fit.)"""
    import torch
    from pyflac_amd import batch
    from oracle import oracle as O
    monkeypatch.setenv('FLACGPU_FBW', '28')
    monkeypatch.setenv('FLACGPU_DIRECT24', '0')          # (the chunk form: the direct form has one frame buffer, no windows)
    rng = np.random.default_rng(11)
    bs = 4096
    t = np.arange(bs)
    tone = lambda a, f, ph: np.round(a * np.sin(2 * np.pi * f * t / 48000 + ph) + rng.normal(0, a / 300, bs)).astype(np.int64)
    blocks = [np.stack([tone(3e6, 440 + 10 * k, 0), tone(2e6, 660, k)], axis=1) << 8 for k in range(6)]
    blocks.insert(3, rng.integers(-2**31, 2**31, (bs, 2)))                       # noise over the whole range: verbatim subframes
    blocks.append(rng.integers(-2**31, 2**31, (777, 2)))                         # a true 32-bit ragged tail (short lanes: it fits)
    arr = np.concatenate(blocks).astype(np.int32)
    s = batch.settings(5, 2, 32, 48000, bs, True)
    cfg, _ = O.config(5, 2, 32, 48000, bs, True)
    want, sizes = O.encode_stream(cfg, arr)
    dev = torch.from_numpy(arr).cuda()
    got = []
    for timing in (0, 1, 0):
        c = batch.Context(0, testhooks=True)
        L = c._L
        L.flacgpu_set_log_guard(c._h, 1e30)              # (every order guess counts as a near tie: the counters are busy)
        L.flacgpu_set_stage_timing(c._h, timing)
        for _rep in range(2):                            # (the second call starts from counters the first one's signal kernel left)
            out, offs, st = c.encode(s, dev)
            assert st.redo_blocks == 1
            got.append((st.log_guard_subframes, st.lpc_order_min_margin, bytes(out[:st.total_bytes].cpu().numpy().tobytes())))
        c.close()
    assert got[0][2] == want[len(want) - int(sizes.sum()):]
    assert got[0][0] > 0 and np.isfinite(got[0][1])
    assert all(g == got[0] for g in got)


def test_limit_min_bitrate_and_a_constant_left_channel_of_28_bits_and_more(ctx):
    """limit_min_bitrate disables CONSTANT for the last independent channel (and then for mid and side) when every earlier channel
    CHOSE CONSTANT -- and from 28 bits per sample on libFLAC's order guess (the _limit_residual forms) flags only an all-zero signal
    as constant: a 32-bit stream at a non-zero DC level keeps its CONSTANT mid channel, one whose channels are equal its CONSTANT
    side channel.  (gpu_fuzz seeds 415128 and 410060 of round 4: the pipeline looked at the samples of the left channel instead of
    at what the left channel's subframe would be.)"""
    import torch
    from pyflac_amd import batch
    from oracle import oracle as O
    n = 4608 * 3 + 1000
    dc = np.stack([np.full(n, 1540236309, np.int64), np.full(n, 88344043, np.int64)], axis=1)
    eq = np.stack([np.full(n, 932007123, np.int64), np.full(n, 932007123, np.int64)], axis=1)
    zl = np.stack([np.zeros(n, np.int64), np.full(n, 88344043, np.int64)], axis=1)              # an all-zero left channel IS constant
    w5 = np.stack([np.full(n, 1540236309 & ~63, np.int64), np.full(n, 88344043, np.int64)], axis=1)   # six wasted bits: 26 bits, constant
    for arr64 in (dc, eq, zl, w5):
        arr = arr64.astype(np.int32)
        for level, bs in ((6, 4608), (8, 2048)):
            s = batch.settings(level, 2, 32, 96000, bs, True)
            cfg, _ = O.config(level, 2, 32, 96000, bs, True)
            s.limit_min_bitrate = 1
            cfg.limit_min_bitrate = 1
            out, offs, st = ctx.encode(s, torch.from_numpy(arr).cuda())
            want, sizes = O.encode_stream(cfg, arr)
            assert out[:st.total_bytes].cpu().numpy().tobytes() == want[86:], (level, bs)


def test_32_bit_mono_and_many_channels_with_shared_wasted_bits(ctx):
    import torch
    from pyflac_amd import batch
    from oracle import oracle as O
    for channels in (1, 3):
        pcm = _multichannel_pcm(7 + channels, channels, 4096 * 3 + 100, 24)
        arr = _in32(pcm)
        s = batch.settings(5, channels, 32, 48000, 4096, True)
        cfg, _ = O.config(5, channels, 32, 48000, 4096, True)
        out, offs, st = ctx.encode(s, torch.from_numpy(arr).cuda())
        want, sizes = O.encode_stream(cfg, arr)
        assert out[:st.total_bytes].cpu().numpy().tobytes() == want[86:]


def test_matrix_core_selfcheck_and_its_fallback(golden):
    """flacgpu_ctx_create checks that v_mfma_f64_4x4x4_4b_f64 sums like a chain of v_fma_f64 -- what the bit-exactness of the
    pipeline's autocorrelation rests on -- with random operands against the VALU chain.  On the MI355X the count of
    differing results is 0.  A device where it is not keeps the bytes: every block then takes the generic kernel, and the context
    says so (the outcome is overridden here to drive that path)."""
    from pyflac_amd import batch, _lib
    L = _lib.lib()
    c = batch.Context(0)
    note = C.c_char_p()
    assert L.flacgpu_selfcheck(c._h, C.byref(note)) == 0 and note.value == b''
    names = ('cfg2_20s_l5', 'cfg4_10s_l8')

    def encode_all():
        out = {}
        for name in names:
            spec, sr, level, bs, subset = cases.ENCODE_CASES[name]
            pcm, bps = cases.make_pcm(spec)
            stream, _offs, _s = _gpu_stream(c, cases.as_int_array(pcm, bps), sr, bps, level, bs, subset)
            out[name] = hashlib.sha256(stream).hexdigest()
        return out
    want = {n: golden[n]['sha256'] for n in names}
    assert encode_all() == want
    L.flacgpu_force_selfcheck_result(c._h, 7)
    assert L.flacgpu_selfcheck(c._h, C.byref(note)) == 7 and b'generic kernel' in note.value
    assert encode_all() == want                   # same bytes through the generic kernel
    L.flacgpu_force_selfcheck_result(c._h, 0)
    assert L.flacgpu_selfcheck(c._h, C.byref(note)) == 0
    assert encode_all() == want


_QUICK_SCRIPT = r'''
import sys, hashlib, json
import numpy as np, torch
sys.path.insert(0, %r)
from pyflac_amd import batch, synth
ctx = batch.Context(0)
pcm = synth.config2_stereo16(100.0, 5)[:4608 * 1024]
t = torch.from_numpy(pcm.astype(np.int32)).cuda()
res = []
for level, bs in ((5, 1024), (5, 1024), (5, 1024), (8, 1024), (5, 1024)):          # (repeated layouts: the second call of a layout starts quick)
    s = batch.settings(level, 2, 16, 48000, bs, True)
    out, offs, st = ctx.encode(s, t)
    res.append([hashlib.sha256(out[:st.total_bytes].cpu().numpy().tobytes()).hexdigest(), int(st.nblocks), int(st.log_guard_subframes),
                float(st.lpc_order_min_margin), int(st.error_flags)])
print('RESULT ' + json.dumps(res))
'''


def test_grouped_launch_starts_the_same_with_and_without_its_begin_kernel():
    """Round 4: a launch of several groups (4096 blocks and more) starts without fg_pipe_begin_kernel and without the fork event when
    the previous call's signal kernel left the guard counters reset and the block list is the last call's (FgPipeLaunch.guard_clean,
    no_fork).  Same bytes and the same guard statistics as with the begin kernel in front of every launch (FLACGPU_QUICK_START=0, a
    child process each), over repeated and changing layouts -- and the first stream equals the oracle's."""
    import json, subprocess, sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    outs = []
    for v in ('1', '0'):
        env = dict(os.environ, FLACGPU_QUICK_START=v, PYFLAC_AMD_TESTHOOKS='1')       # (the selector is read by the test-hooks build only)
        p = subprocess.run([sys.executable, '-c', _QUICK_SCRIPT % root], env=env, capture_output=True, text=True, timeout=900)
        assert p.returncode == 0, p.stderr[-2000:]
        line = [l for l in p.stdout.splitlines() if l.startswith('RESULT ')][-1]
        outs.append(json.loads(line[7:]))
    assert outs[0] == outs[1]
    assert outs[0][0] == outs[0][1] == outs[0][2] == outs[0][4] and outs[0][0][1] >= 4096 and outs[0][0][4] == 0
    from pyflac_amd import synth
    from oracle import oracle as O
    pcm = synth.config2_stereo16(100.0, 5)[:4608 * 1024]
    cfg, _ = O.config(5, 2, 16, 48000, 1024, True)
    want, sizes = O.encode_stream(cfg, pcm.astype(np.int32))
    import hashlib
    assert hashlib.sha256(want[86:]).hexdigest() == outs[0][0][0]
