"""Build recipe for libff3d_hip.so (gfx950 only).  hipcc cross-compiles without a GPU.

    python -m focalformer3d_amd.build          # rebuild what is stale
    python -m focalformer3d_amd.build --force  # rebuild everything

Incremental: every csrc/*.hip is compiled to its own object under lib/obj/ (in parallel, only when the source or a
header is newer than the object), then linked into focalformer3d_amd/lib/libff3d_hip.so (in-tree, so the built library
travels with the repo snapshot to the GPU box).
"""
import glob
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
LIB_DIR = os.path.join(PKG, 'lib')
# FF3D_BUILD_EXPERIMENTS=1 builds a SECOND library next to the shipped one (lib/libff3d_hip_exp.so, objects in lib/obj_exp):
# A/B sessions select it with FF3D_LIB=<path>; the product never loads it by default.
_EXP = os.environ.get('FF3D_BUILD_EXPERIMENTS') == '1'
OBJ_DIR = os.path.join(LIB_DIR, 'obj_exp' if _EXP else 'obj')
LIB_PATH = os.path.join(LIB_DIR, 'libff3d_hip_exp.so' if _EXP else 'libff3d_hip.so')
SOURCES = sorted(glob.glob(os.path.join(PKG, 'csrc', '*.hip')))
HEADERS = sorted(glob.glob(os.path.join(PKG, 'csrc', '*.h'))) + [os.path.join(ROOT, 'include', 'ff3d.h')]
# packed fp32 instructions are off: some of their forms have given wrong results on these cards (the host pass warns that it does not
# know the feature)
CFLAGS = ['--offload-arch=gfx950', '-O3', '-std=c++17', '-fPIC', '-Xclang', '-target-feature', '-Xclang', '-packed-fp32-ops',
          '-I' + os.path.join(ROOT, 'include')]
# FF3D_BUILD_EXPERIMENTS=1: also compile the measured-slower kernel variants and timing ablations that round 1-4's A/B
# records in profiles/ came from (hand-scheduled / 8 x 64 halo convs, 192-column and periodic weight-stationary GEMMs,
# FF3D_HALO_ABLATE / FF3D_WS_ABLATE instances).  The shipped library does not carry them.
EXPERIMENTS = _EXP
if EXPERIMENTS:
    CFLAGS.append('-DFF3D_BUILD_EXPERIMENTS')
FLAGS_STAMP = os.path.join(OBJ_DIR, 'cflags.txt')


def _obj(src):
    return os.path.join(OBJ_DIR, os.path.splitext(os.path.basename(src))[0] + '.o')


def _newer(path, than):
    return (not os.path.exists(path)) or any(os.path.getmtime(f) > os.path.getmtime(path) for f in than)


def _flags_changed():
    try:
        return open(FLAGS_STAMP).read() != ' '.join(CFLAGS)
    except OSError:
        return bool(glob.glob(os.path.join(OBJ_DIR, '*.o')))        # objects of unknown flags


def stale():
    return _newer(LIB_PATH, SOURCES + HEADERS) or _flags_changed()


def build(force=False, verbose=True):
    """Compile every HIP source into focalformer3d_amd/lib/libff3d_hip.so; returns its path."""
    if not force and not stale():
        return LIB_PATH
    hipcc = os.environ.get('HIPCC', '/opt/rocm/bin/hipcc')
    os.makedirs(OBJ_DIR, exist_ok=True)
    force = force or _flags_changed()               # objects built with other flags (experiments on / off) are not reused
    todo = [s for s in SOURCES if force or _newer(_obj(s), [s] + HEADERS)]

    def compile_one(src):
        cmd = [hipcc] + CFLAGS + ['-c', src, '-o', _obj(src)]
        if verbose:
            print(' '.join(cmd), file=sys.stderr)
        subprocess.run(cmd, check=True)

    with ThreadPoolExecutor(max_workers=max(1, min(len(todo), os.cpu_count() or 1))) as ex:
        list(ex.map(compile_one, todo))
    known = {_obj(s) for s in SOURCES}
    for stray in glob.glob(os.path.join(OBJ_DIR, '*.o')):       # objects of deleted sources must not be linked
        if stray not in known:
            os.remove(stray)
    cmd = [hipcc, '--offload-arch=gfx950', '-shared', '-fPIC'] + sorted(known) + ['-o', LIB_PATH]
    if verbose:
        print(' '.join(cmd), file=sys.stderr)
    subprocess.run(cmd, check=True)
    with open(FLAGS_STAMP, 'w') as f:
        f.write(' '.join(CFLAGS))
    return LIB_PATH


if __name__ == '__main__':
    build(force='--force' in sys.argv)
