"""build(): the product library is compiled, linked and loaded whatever becomes of the emulator that the CPU tests run on, and a library that
other sources made is found out. The compilers are stand-ins here: one writes empty objects and, asked to link, hands out the library that
is there; the other fails."""
import shutil
import subprocess

import pytest

import __graft_entry__ as entry


def script(path, text):
    path.write_text('#!/bin/sh\n' + text)
    path.chmod(0o755)
    return str(path)


@pytest.fixture
def build_in(tmp_path, monkeypatch):
    """build() with its outputs under tmp_path and the given stand-in compilers"""
    if not entry.HIP_LIB.exists():
        pytest.skip('no product library to hand out')
    built = tmp_path / 'prebuilt.so'
    shutil.copy(entry.HIP_LIB, built)
    good = script(tmp_path / 'good', f'for a in "$@"; do last=$a; done\ncase " $* " in *" -shared "*) cp {built} "$last";; *) : > "$last";; esac\n')
    bad = script(tmp_path / 'bad', 'exit 1\n')
    for name, at in (('OBJ', 'obj'), ('HIP_LIB', 'product.so'), ('EMU_LIB', 'emulator.so')):
        monkeypatch.setattr(entry, name, tmp_path / at)

    def run(hipcc, hostcxx):
        monkeypatch.setenv('HIPCC', {'good': good, 'bad': bad}[hipcc])
        monkeypatch.setenv('HOSTCXX', {'good': good, 'bad': bad}[hostcxx])
        entry.build()
    run.dir = tmp_path
    return run


def test_a_failing_emulator_leaves_a_whole_product(build_in):
    with pytest.warns(RuntimeWarning, match='emulator'):
        build_in('good', 'bad')
    assert (build_in.dir / 'product.so').exists() and not (build_in.dir / 'emulator.so').exists()


def test_a_failing_product_is_an_error(build_in):
    with pytest.raises(subprocess.CalledProcessError):
        build_in('bad', 'good')
    assert not (build_in.dir / 'product.so').exists()


def test_both_are_built(build_in, recwarn):
    build_in('good', 'good')
    assert (build_in.dir / 'product.so').exists() and (build_in.dir / 'emulator.so').exists()
    assert not [w for w in recwarn if 'emulator' in str(w.message)]


@pytest.mark.parametrize('lib', ['EMU_LIB', pytest.param('HIP_LIB', marks=pytest.mark.gpu)])
def test_the_library_under_test_is_that_of_the_sources(lib):
    current = entry.is_current(getattr(entry, lib))
    if current is None:
        pytest.skip('the library carries no hash of its sources')
    assert current, 'a source was changed after the library was built: call __graft_entry__.build()'


def test_a_changed_source_is_found_out(build_in, monkeypatch):
    """any kernel, the ABI and, for the emulator, its own sources; a library without its hash is of unknown sources"""
    src = build_in.dir / 'tree'
    for d in ('gigagan_pytorch_amd/csrc', 'include', 'tests/emu'):
        shutil.copytree(entry.ROOT / d, src / d, ignore=shutil.ignore_patterns('*.so', '*.sources'))
    build_in('good', 'good')
    monkeypatch.setattr(entry, 'ROOT', src)
    monkeypatch.setattr(entry, 'CSRC', src / 'gigagan_pytorch_amd' / 'csrc')
    assert entry.is_current(entry.HIP_LIB) and entry.is_current(entry.EMU_LIB)
    changed = src / 'tests' / 'emu' / 'gg_device_emu.h'
    changed.write_text(changed.read_text() + '//')
    assert entry.is_current(entry.HIP_LIB) and entry.is_current(entry.EMU_LIB) is False
    changed = src / 'gigagan_pytorch_amd' / 'csrc' / 'gg_window.h'
    changed.write_text(changed.read_text() + '//')
    assert entry.is_current(entry.HIP_LIB) is False
    entry.HIP_LIB.with_suffix('.so.sources').unlink()
    assert entry.is_current(entry.HIP_LIB) is None
