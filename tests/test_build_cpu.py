"""CPU: build fingerprints, and what is attached to or loaded with a library by them."""
import json
import os
import shutil
import subprocess
import sys

import pytest

import bench
from conftest import REPO
from minitchess_alphazero_amd import build


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """A copy of the library's sources that build.py's fingerprints are taken of."""
    shutil.copytree(build.CSRC, tmp_path / 'csrc')
    shutil.copytree(build.INCLUDE, tmp_path / 'include')
    monkeypatch.setattr(build, 'CSRC', str(tmp_path / 'csrc'))
    monkeypatch.setattr(build, 'INCLUDE', str(tmp_path / 'include'))
    return tmp_path


def append(path, text):
    with open(path, 'a') as f:
        f.write(text)


def test_engine_hash_is_the_engines_alone(tree):
    first, whole = build.engine_hash(), build.source_hash()
    for name in build.OPERATOR_FILES:
        append(tree / 'csrc' / name, '// changed\n')
    header = (tree / 'include' / 'mtaz.h').read_text()
    (tree / 'include' / 'mtaz.h').write_text(header.replace('int mtaz_muon_step(int device', 'int mtaz_muon_step(int dev'))
    assert build.engine_hash() == first and build.source_hash() != whole
    for path in ('csrc/mtaz_net16.hip', 'csrc/engine.h', 'csrc/mtaz_host.cpp', 'include/mtaz.h'):
        before = build.engine_hash()
        append(tree / path, '// changed\n')
        assert build.engine_hash() != before, path


def test_traffic_stays_attached_while_only_operators_change(tree):
    path = str(tree / 'traffic.json')
    passes = {'kernel': 'k_net_y', 'games': 4096, 'sims': 64, 'hbm_bytes_per_launch': 8.5e8, 'engine_sha256': build.engine_hash()}
    with open(path, 'w') as f:
        json.dump(passes, f)
    append(tree / 'csrc' / 'mtaz_muon.hip', '// changed\n')
    assert bench.traffic_of(path, build.engine_hash(), 4096, 64, 'k_net_y (fused)')[0] == 8.5e8
    for games, sims, kernel in ((2048, 64, 'k_net_y'), (4096, 36, 'k_net_y'), (4096, 64, 'k_net_z')):
        traffic, why = bench.traffic_of(path, build.engine_hash(), games, sims, kernel)
        assert traffic is None and 'another workload' in why
    append(tree / 'csrc' / 'mtaz_net16.hip', '// changed\n')
    traffic, why = bench.traffic_of(path, build.engine_hash(), 4096, 64, 'k_net_y (fused)')
    assert traffic is None and why.startswith('stale')
    assert bench.traffic_of(os.path.join(str(tree), 'none.json'), '', 4096, 64, 'k_net_y')[0] is None


def test_built_libraries_are_not_built_again(monkeypatch):
    """Both libraries carry the fingerprint of what they are built from where it is looked for."""
    assert build.embedded_hash(build.OUT_AUTOGRAD, b'mtaz-autograd-sha256=') == build.autograd_hash()

    def command(*args, **kwargs):
        raise AssertionError(f'a compiler was called: {args}')
    monkeypatch.setattr(build.subprocess, 'check_call', command)
    monkeypatch.setattr(build.subprocess, 'Popen', command)
    assert build.build(verbose=False) == build.OUT


def test_autograd_hash_covers_the_compile_command(monkeypatch):
    first = build.autograd_hash()
    monkeypatch.setattr(build, 'AUTOGRAD_FLAGS', build.AUTOGRAD_FLAGS + ['-DX'])
    assert build.autograd_hash() != first


def test_another_library_is_the_only_one_loaded(tmp_path):
    """MTAZ_LIB names another file: the operators of libmtaz_autograd.so call that one too."""
    other = tmp_path / 'another_build.so'
    shutil.copy(build.OUT, other)
    code = ('from minitchess_alphazero_amd import _lib\n'
            '_lib.nodes()\n'
            'print(sorted({l.split()[-1] for l in open("/proc/self/maps") if "libmtaz.so" in l or "another_build" in l}))')
    out = subprocess.run([sys.executable, '-c', code], env={**os.environ, 'MTAZ_LIB': str(other)}, cwd=REPO, check=True,
                         capture_output=True, text=True).stdout
    assert out.strip().splitlines()[-1] == str([str(other)])
