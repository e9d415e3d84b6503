"""A build that is not forced compiles what is out of date: sources, headers, and objects that another command line made."""
import os
import stat

from deepwmh_amd import build


def test_objects_made_with_other_flags_are_compiled_again(tmp_path, monkeypatch):
    csrc, lib, log = tmp_path / 'deepwmh_amd' / 'csrc', tmp_path / 'deepwmh_amd' / 'lib', tmp_path / 'log'
    csrc.mkdir(parents=True)
    (tmp_path / 'include').mkdir()
    for name in ('a.hip', 'b.hip', 'wmh_common.h', 'conv3d_common.h', 'cl_common.h', 'act8_common.h'):
        (csrc / name).write_text('')
    (tmp_path / 'include' / 'deepwmh_amd.h').write_text('')
    cc = tmp_path / 'cc'
    cc.write_text('#!/bin/sh\necho "$@" >> %s\nfor last; do :; done\ncase "$*" in *-shared*) exit 0;; *) : > "$last";; esac\n' % log)
    cc.chmod(cc.stat().st_mode | stat.S_IXUSR)
    for name, value in (('HERE', str(tmp_path / 'deepwmh_amd')), ('CSRC', str(csrc)), ('LIBDIR', str(lib)), ('HIPCC', str(cc)), ('SOURCES', ['a.hip', 'b.hip']),
                        ('FLAGS', ['-O3'])):
        monkeypatch.setattr(build, name, value)
    out = str(lib / 'lib.so')

    def compiled(extra=()):
        log.write_text('')
        build._build_one(out, 'obj', list(extra), False, False)
        open(out, 'w').close()
        lines = log.read_text().splitlines()
        units = sorted(os.path.basename(line.split(' -o ')[1])[:-2] for line in lines if '-shared' not in line)
        assert ('-shared' in ''.join(lines)) == bool(units)     # linked again where something was compiled
        return units
    assert compiled() == ['a', 'b']
    assert compiled() == []
    assert compiled(['-DWMH_DIAG']) == ['a', 'b'] and compiled(['-DWMH_DIAG']) == []
    assert compiled() == ['a', 'b'] and compiled() == []
    monkeypatch.setattr(build, 'FLAGS', ['-O3', '-Xclang', '-target-feature', '-Xclang', '-packed-fp32-ops'])
    assert compiled() == ['a', 'b'] and compiled() == []
    os.remove(out)                                              # (a link that failed, or one of older objects)
    log.write_text('')
    build._build_one(out, 'obj', [], False, False)
    assert '-shared' in log.read_text()
    open(out, 'w').close()
    os.utime(out, (1, 1))
    log.write_text('')
    build._build_one(out, 'obj', [], False, False)
    assert '-shared' in log.read_text()
    os.remove(str(lib / 'obj' / 'b.cmd'))                       # (of a build that did not note it)
    assert compiled() == ['b'] and compiled() == []
