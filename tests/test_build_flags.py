"""The build's command lines (no compiler needed): every translation unit with its own flags, the measurement aid with the same ones."""
import inspect
import os
import stat
import subprocess

import pytest

import __graft_entry__ as graft

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_build_takes_what_it_took():
    assert [p.default is not inspect.Parameter.empty for p in inspect.signature(graft.build).parameters.values()] == [True]
    assert 'force' in inspect.signature(graft.build).parameters


@pytest.mark.parametrize('unit', ['libfmarl', 'fmarl_memory', 'fmarl_block', 'fmarl_actions'])
def test_the_measurement_aid_compiles_what_is_built(unit, tmp_path):
    assert unit in graft.UNITS and os.path.exists(os.path.join(graft.CSRC, unit + '.hip'))
    seen, stub = tmp_path / 'args', tmp_path / 'hipcc'
    stub.write_text('#!/bin/sh\nfor a in "$@"; do echo "$a"; done > %s\n' % seen)
    stub.chmod(stub.stat().st_mode | stat.S_IXUSR)
    subprocess.check_call(['bash', os.path.join(ROOT, 'tools', 'kres.sh'), unit], env=dict(os.environ, HIPCC=str(stub)))
    args = seen.read_text().split('\n')
    assert args[:len(graft.flags(unit))] == graft.flags(unit) and unit + '.hip' in args
    assert ('-ffp-contract=off' in args) == (unit == 'libfmarl')
