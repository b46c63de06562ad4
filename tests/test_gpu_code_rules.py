"""
What the GPU code of this repository may hold, checked over its sources: the kernels, the headers they include, the probes
under tools/ and every script that could build one.
"""

import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOURCE_DIRS = ('nufhe_amd', 'nufhe', 'include', 'tools', 'examples', 'oracle', 'tests')
SOURCE_TYPES = ('.hip', '.h', '.hpp', '.c', '.cpp', '.s', '.S', '.py', '.sh')

# stores and atomics of the scalar unit, and that cache's write-back and discard
SCALAR_WRITE = re.compile(r'\bs_(?:(?:buffer_|scratch_)?store_|(?:buffer_)?atomic_|dcache_(?:wb|discard))')

# the vector unit's packed FP32 arithmetic: some of its forms have given wrong results now and then, with no error
PACKED_FP32 = re.compile(r'\bv_pk_(?:add|mul|fma)_f32')


def sources():
    for top in SOURCE_DIRS:
        for where, dirs, files in os.walk(os.path.join(ROOT, top)):
            dirs[:] = [d for d in dirs if d not in ('__pycache__', 'build', '_ref')]
            for name in files:
                if name.endswith(SOURCE_TYPES) or name == 'Makefile':
                    yield os.path.join(where, name)


def hits(pattern):
    found = []
    for path in sources():
        with open(path, errors='replace') as f:
            for number, line in enumerate(f, 1):
                if pattern.search(line):
                    found.append('%s:%d: %s' % (os.path.relpath(path, ROOT), number, line.strip()))
    return found


def test_the_scan_reaches_the_kernels():
    names = {os.path.relpath(p, ROOT) for p in sources()}
    assert {'nufhe_amd/csrc/kernels.hip', 'nufhe_amd/csrc/api.hip', 'nufhe_amd/csrc/Makefile',
            'tools/microbench_issue.hip', 'tools/build_variant.sh'} <= names


@pytest.mark.parametrize('op', ['store_dword', 'store_dwordx4', 'buffer_store_dword', 'scratch_store_dword', 'atomic_add',
                                'buffer_atomic_add', 'dcache_wb', 'dcache_wb_vol', 'dcache_discard'])
def test_the_pattern_knows_the_scalar_writes(op):
    assert SCALAR_WRITE.search('asm volatile("s_%s s0, s[2:3], 0")' % op)


@pytest.mark.parametrize('op', ['load_dwordx2', 'buffer_load_dword', 'dcache_inv', 'waitcnt'])
def test_the_pattern_leaves_the_reads_alone(op):
    assert not SCALAR_WRITE.search('asm volatile("s_%s s0, s[2:3], 0")' % op)


def test_no_write_through_the_scalar_data_cache():
    """GPU memory is written with vector stores: nothing writes the scalar data cache back on its own, and the unit's own
    write-back is no part of this code."""
    assert hits(SCALAR_WRITE) == []


@pytest.mark.parametrize('op', ['add_f32', 'mul_f32', 'fma_f32'])
def test_the_pattern_knows_the_packed_fp32_arithmetic(op):
    assert PACKED_FP32.search('asm volatile("v_pk_%s v[0:1], v[0:1], v[2:3]")' % op)


@pytest.mark.parametrize('op', ['add_u16', 'fma_f16', 'mul_lo_u16'])
def test_the_pattern_leaves_the_16_bit_packed_arithmetic_alone(op):
    assert not PACKED_FP32.search('asm volatile("v_pk_%s v0, v0, v1")' % op)


def test_no_packed_fp32_arithmetic_by_hand():
    assert hits(PACKED_FP32) == []


NO_PACKED_FP32 = '-Xclang -target-feature -Xclang -packed-fp32-ops'


def library_compiles(*make_args):
    """the compile commands `make` would run for the library's objects"""
    text = subprocess.run(['make', '-n'] + list(make_args), cwd=os.path.join(ROOT, 'nufhe_amd', 'csrc'), text=True, check=True,
                          capture_output=True).stdout
    return [l for l in text.split('\n') if ' -c ' in l]


def test_every_object_is_compiled_without_packed_fp32():
    lines = library_compiles('-B')
    assert len(lines) == 5 and all(NO_PACKED_FP32 in l for l in lines)


def test_other_flags_make_other_objects(tmp_path):
    """An object that is older than the Makefile is compiled again: it may have been made with other flags."""
    csrc = tmp_path / 'nufhe_amd' / 'csrc'
    shutil.copytree(os.path.join(ROOT, 'nufhe_amd', 'csrc'), csrc, ignore=shutil.ignore_patterns('*.o'))
    shutil.copytree(os.path.join(ROOT, 'include'), tmp_path / 'include')
    objects = ['kernels.o', 'kernels_team8.o', 'kernels_team.o', 'kernels_xfft.o', 'api.o']
    for name in objects:
        (csrc / name).touch()
    times = {name: 2000 for name in objects}
    for makefile, compiled in ((1000, 0), (3000, len(objects))):
        times['Makefile'] = makefile
        for path in list(csrc.iterdir()) + list((tmp_path / 'include').iterdir()):
            os.utime(path, (times.get(path.name, 1000),) * 2)
        out = subprocess.run(['make', '-n'] + objects, cwd=csrc, text=True, check=True, capture_output=True).stdout
        assert sum(' -c ' in l for l in out.split('\n')) == compiled


def test_scripts_compile_without_packed_fp32_too():
    """The tools that build variants of the library, read its ISA or say how a probe is built."""
    for path in sources():
        with open(path, errors='replace') as f:
            text = f.read()
        if os.path.basename(os.path.dirname(path)) == 'tools' and re.search(r"hipcc\b.*offload-arch|hipcc \$FLAGS", text):
            assert NO_PACKED_FP32 in text or NO_PACKED_FP32.replace(' ', "', '") in text, path


def test_the_flags_keep_packed_fp32_out_of_the_isa(tmp_path):
    """Float code that the compiler would pair by itself: packed arithmetic without the flags, none with the library's."""
    src = tmp_path / 'pairs.hip'
    src.write_text('#include <hip/hip_runtime.h>\n'
                   '__global__ void k(float2 *x, float2 a, float2 b)\n'
                   '{ float2 v = x[threadIdx.x]; v.x = v.x * a.x + b.x; v.y = v.y * a.y + b.y; x[threadIdx.x] = v; }\n')
    with_flags = library_compiles('-B')[0].split(' -c ')[0].split()
    plain = [w for w in with_flags if w not in NO_PACKED_FP32.split()]
    found = {}
    for name, cmd in (('flags', with_flags), ('plain', plain)):
        out = tmp_path / (name + '.s')
        subprocess.check_call(cmd + ['--cuda-device-only', '-S', str(src), '-o', str(out)], stderr=subprocess.DEVNULL)
        found[name] = bool(PACKED_FP32.search(out.read_text()))
    assert found == {'flags': False, 'plain': True}


def test_build_compiles_what_is_already_built(monkeypatch):
    """build() is the check that the sources compile: it runs the compiler on every unit, whatever objects are there."""
    import __graft_entry__
    run = []
    monkeypatch.setattr(__graft_entry__.subprocess, 'check_call', lambda cmd, **kw: run.append(cmd))
    __graft_entry__.build()
    library = [cmd for cmd in run if any(str(w).endswith(os.path.join('nufhe_amd', 'csrc')) for w in cmd)]
    assert len(library) == 1
    text = subprocess.run(library[0] + ['-n'], text=True, check=True, capture_output=True).stdout
    assert sum(' -c ' in l for l in text.split('\n')) == 5
