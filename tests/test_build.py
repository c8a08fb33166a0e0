"""build(): the product library is compiled, linked and loaded whatever becomes of the emulator that the CPU tests run on. The compilers
are stand-ins here: one writes empty objects and, asked to link, hands out the library that is there; the other fails."""
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
