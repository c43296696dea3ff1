"""csrc/build.py: the library does not need torch, the autograd nodes' file is made beside it where there is one."""
import subprocess

import pytest

from trajnetplusplusbaselines_amd.csrc import build


@pytest.fixture
def commands(monkeypatch, tmp_path):
    """what build() runs, nothing of it carried out; a test says which command fails"""
    ran = []

    def call(cmd):
        ran.append(cmd)
        if call.fails and call.fails in ' '.join(cmd):
            raise subprocess.CalledProcessError(1, cmd)

    call.fails = None
    monkeypatch.setattr(build.subprocess, 'check_call', call)
    for name in ('OUT_DIR', 'OUT', 'TORCH_OUT'):
        monkeypatch.setattr(build, name, str(tmp_path / getattr(build, name).rsplit('/', 1)[1]))
    return ran, call


def _links(ran):
    return [c for c in ran if build.OUT in c]


def test_the_library_is_made_without_torch(commands, monkeypatch):
    ran, _ = commands
    monkeypatch.setattr(build.importlib.util, 'find_spec', lambda name: None)
    assert build.build(force=True) == build.OUT
    assert len(_links(ran)) == 1 and not any(build.TORCH_SOURCE in ' '.join(c) for c in ran)


def test_the_library_is_made_beside_a_torch_without_rocm(commands, monkeypatch, tmp_path):
    ran, _ = commands
    (tmp_path / 'torch' / 'lib').mkdir(parents=True)
    spec = type('Spec', (), {'submodule_search_locations': [str(tmp_path / 'torch')]})
    monkeypatch.setattr(build.importlib.util, 'find_spec', lambda name: spec)
    build.build(force=True)
    assert len(_links(ran)) == 1 and not any(build.TORCH_SOURCE in ' '.join(c) for c in ran)


def test_the_library_is_made_though_the_torch_file_fails(commands):
    ran, call = commands
    call.fails = build.TORCH_SOURCE
    with pytest.raises(subprocess.CalledProcessError):
        build.build(force=True)
    assert len(_links(ran)) == 1


def test_the_torch_file_is_compiled_with_its_warnings(commands):
    ran, _ = commands
    build.build(force=True)
    cmd, = [c for c in ran if any(a.endswith(build.TORCH_SOURCE) for a in c)]
    assert '-Wall' in cmd and '-w' not in cmd
