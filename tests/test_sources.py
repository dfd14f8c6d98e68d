"""What the sources of this repository do not hold."""
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
KINDS = ('.h', '.c', '.cpp', '.hip', '.inc', '.s', '.py', '.sh')


def _sources():
    for base, dirs, files in os.walk(ROOT):
        dirs[:] = [d for d in dirs if not d.startswith(('.', '_')) and d not in ('gpurun_out', 'golden')]
        for f in files:
            if f.endswith(KINDS) or f == 'Makefile':
                yield os.path.join(base, f)


def _holders(pattern):
    rx = re.compile(pattern)
    out = []
    for path in _sources():
        with open(path, errors='replace') as f:
            out += ['%s:%d' % (os.path.relpath(path, ROOT), i) for i, line in enumerate(f, 1) if rx.search(line)]
    return out


def test_the_walk_finds_the_sources():
    names = {os.path.relpath(p, ROOT) for p in _sources()}
    assert {'bench.py', 'tests/emu/emu.h', 'pyflac_amd/csrc/flac_enc_pipe_impl.h', 'pyflac_amd/csrc/Makefile'} <= names


@pytest.mark.parametrize('pattern', [
    r'\bs_(scratch_|buffer_)?' + r'store_' + r'dword', r'\bs_(buffer_)?' + r'atomic_', r's_dcache' + r'_(wb|discard)'])
def test_nothing_writes_through_the_scalar_data_cache(pattern):
    """No kernel here does, and the emulator's opcode table does not know such an instruction: it would report one as unknown."""
    assert _holders(pattern) == []


@pytest.mark.parametrize('pattern', ['FLACGPU_' + 'STOP', 'FGX_' + 'DBG'])
def test_no_switch_ends_a_launch_after_a_stage(pattern):
    assert _holders(pattern) == []


def test_no_source_names_a_prebuilt_library_of_the_reference():
    assert _holders(r'lib' + r'FLAC[-\d.]*\.(so|dll|dylib)') == []
