"""When build() compiles: a missing object, a newer source or header, other flags; nothing otherwise."""
import os
import types

import pytest

from semseg_amd import build


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """two sources, a header and the host module; commands are noted, not run: they leave the file they were to make"""
    csrc = tmp_path / 'csrc'
    csrc.mkdir()
    for name in ('a.hip', 'b.hip', 'c.h', 'native.cpp'):
        (csrc / name).write_text('')
        os.utime(csrc / name, (1, 1))
    for name, path in (('CSRC', csrc), ('OBJ', csrc / 'build'), ('LIB', tmp_path / 'lib.so'), ('NATIVE', tmp_path / 'native.so')):
        monkeypatch.setattr(build, name, str(path))
    monkeypatch.setattr(build, 'native_command', lambda: ['g++', '-O2', str(csrc / 'native.cpp'), '-o', str(tmp_path / 'native.so')])
    t = types.SimpleNamespace(csrc=csrc, commands=[], fail=False)

    def run(cmd, **kw):
        t.commands.append(cmd)
        if not t.fail:
            open(cmd[cmd.index('-o') + 1], 'w').close()
        return types.SimpleNamespace(returncode=int(t.fail), stderr='failed')
    monkeypatch.setattr(build.subprocess, 'run', run)

    def made():
        t.commands.clear()
        build.build(verbose=False)
        return sorted(os.path.basename(c[c.index('-o') + 1]) for c in t.commands)
    t.made = made
    return t


def test_nothing_is_compiled_twice(tree):
    assert tree.made() == ['a.o', 'b.o', 'lib.so', 'native.so']
    assert tree.made() == []
    os.utime(tree.csrc / 'a.hip')
    assert tree.made() in ([], ['a.o', 'lib.so'])              # within a tick of the file system's clock
    os.utime(tree.csrc / 'a.hip', (4e9, 4e9))
    assert tree.made() == ['a.o', 'lib.so']


def test_other_flags_compile_everything_again(tree, monkeypatch):
    tree.made()
    monkeypatch.setattr(build, 'FLAGS', build.FLAGS + ['-DX'])
    assert tree.made() == ['a.o', 'b.o', 'lib.so']
    assert tree.made() == []


def test_another_host_command_compiles_the_host_module_again(tree, monkeypatch):
    tree.made()
    old = build.native_command()
    monkeypatch.setattr(build, 'native_command', lambda: old[:1] + ['-O3'] + old[2:])
    assert tree.made() == ['native.so']
    assert tree.made() == []


def test_an_object_of_unknown_flags_is_compiled_again(tree):
    """a tree that was built before the commands were noted"""
    tree.made()
    for f in (tree.csrc / 'build').glob('*.command'):
        f.unlink()
    assert tree.made() == ['a.o', 'b.o', 'lib.so', 'native.so']


def test_a_failed_command_is_run_again(tree, monkeypatch):
    tree.made()
    monkeypatch.setattr(build, 'FLAGS', build.FLAGS + ['-DX'])
    tree.fail = True
    with pytest.raises(RuntimeError, match='failed'):
        tree.made()
    tree.fail = False
    assert tree.made() == ['a.o', 'b.o', 'lib.so']


def test_a_library_older_than_its_objects_is_linked_again(tree):
    tree.made()
    os.utime(build.LIB, (2, 2))
    assert tree.made() == ['lib.so']
