"""What the sources of this repository do not hold."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OBJDUMP = '/opt/rocm/lib/llvm/bin/llvm-objdump'
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


def test_packed_fp32_is_neither_written_nor_compiled():
    """Some packed FP32 forms have given wrong results now and then: nothing issues them by hand and the compiler is told not to."""
    assert _holders(r'v_pk_' + r'(add|mul|fma)_f32') == []
    with open(os.path.join(ROOT, 'pyflac_amd', 'csrc', 'Makefile')) as f:
        assert '-Xclang -target-feature -Xclang -packed-fp32-ops' in f.read()


@pytest.mark.skipif(not os.path.exists(OBJDUMP), reason='needs llvm-objdump')
def test_the_built_library_holds_no_packed_fp32(tmp_path):
    """The gfx950 assembly of every code object built here."""
    shutil.copy(os.path.join(ROOT, 'pyflac_amd', 'libflacgpu.so'), tmp_path / 'lib.so')
    subprocess.run([OBJDUMP, '--offloading', 'lib.so'], cwd=tmp_path, check=True, capture_output=True)
    objs = sorted(f for f in os.listdir(tmp_path) if 'gfx950' in f)
    assert len(objs) >= 10
    for o in objs:
        text = subprocess.run([OBJDUMP, '-d', '--no-show-raw-insn', '--mcpu=gfx950', o], cwd=tmp_path, check=True, capture_output=True, text=True).stdout
        assert 's_endpgm' in text and not re.search('v_pk_' + '(add|mul|fma)_f32', text), o


def test_no_build_leftover_is_tracked():
    if not os.path.isdir(os.path.join(ROOT, '.git')):
        pytest.skip('not a checkout')
    p = subprocess.run(['git', 'ls-files'], cwd=ROOT, capture_output=True, text=True)
    if p.returncode:
        pytest.skip('git does not answer here')
    files = p.stdout.split('\n')
    assert [f for f in files if f.endswith(('.tmp', '.o', '.so', '.a', '.pyc'))] == []
