"""Builds semseg_amd/libsemseg_hip.so (gfx950 only) from semseg_amd/csrc/*.hip with hipcc, and semseg_amd/_native.so (host code: the autograd
node and lists whose cost is the host's) from csrc/native.cpp, both in-tree."""
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, 'csrc')
OBJ = os.path.join(HERE, 'csrc', 'build')
LIB = os.path.join(HERE, 'libsemseg_hip.so')
# fast-honor-pragmas: contraction everywhere but where a kernel says `#pragma clang fp contract(off)` (plain `fast` ignores it);
# no packed fp32 instructions (v_pk_add / mul / fma_f32): some of their forms have given wrong results on gfx950
FLAGS = ['--offload-arch=gfx950', '-O3', '-std=c++17', '-fPIC', '-ffp-contract=fast-honor-pragmas', '-Wno-unused-result',
         '-Xclang', '-target-feature', '-Xclang', '-packed-fp32-ops']


NATIVE = os.path.join(HERE, '_native.so')


def native_command():
    """csrc/native.cpp -> _native.so: host code against torch's headers (no device code)"""
    import sysconfig
    import torch
    from torch.utils.cpp_extension import include_paths
    root = os.path.dirname(torch.__file__)
    inc = [f for p in include_paths() + ['/opt/rocm/include'] for f in ('-isystem', p)] + ['-I' + sysconfig.get_paths()['include']]
    return ['g++', '-O2', '-std=c++17', '-fPIC', '-shared', '-D__HIP_PLATFORM_AMD__', '-DUSE_ROCM',
            f'-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}'] + inc + [os.path.join(CSRC, 'native.cpp'), '-o', NATIVE,
            '-L' + os.path.join(root, 'lib'), '-ltorch', '-ltorch_cpu', '-ltorch_hip', '-lc10', '-lc10_hip', '-ltorch_python']


def _stamp(src):
    return os.path.join(OBJ, os.path.basename(src) + '.command')


def _newer(src, dst, deps, command):
    """whether dst has to be made: it is missing, older than a source, or was made by another command (other flags, another torch)"""
    if not os.path.exists(dst):
        return True
    if not os.path.exists(_stamp(src)) or open(_stamp(src)).read() != ' '.join(command):
        return True
    t = os.path.getmtime(dst)
    return any(os.path.getmtime(p) > t for p in [src] + deps)


def build(force=False, verbose=True):
    hipcc = os.environ.get('HIPCC', '/opt/rocm/bin/hipcc')
    os.makedirs(OBJ, exist_ok=True)
    srcs = sorted(f for f in os.listdir(CSRC) if f.endswith('.hip'))
    hdrs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith('.h')]
    jobs = []
    for s in srcs:
        src, obj = os.path.join(CSRC, s), os.path.join(OBJ, s[:-4] + '.o')
        cmd = [hipcc] + FLAGS + ['-c', src, '-o', obj]
        if force or _newer(src, obj, hdrs, cmd):
            jobs.append((src, cmd))

    def cc(job):
        src, cmd = job
        if os.path.exists(_stamp(src)):
            os.remove(_stamp(src))                             # a command that fails or is cut off leaves none
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode == 0:
            with open(_stamp(src), 'w') as f:
                f.write(' '.join(cmd))
        return src, r.returncode, r.stderr

    device_jobs = bool(jobs)
    native, cmd = os.path.join(CSRC, 'native.cpp'), native_command()
    if force or _newer(native, NATIVE, [], cmd):
        jobs.append((native, cmd))
    with ThreadPoolExecutor(max_workers=min(8, max(1, len(jobs)))) as ex:
        for src, rc, err in ex.map(cc, jobs):
            if verbose:
                print(f'[build] {os.path.basename(src)} -> rc {rc}')
            if rc != 0:
                raise RuntimeError(f'compiling {src} failed:\n{err}')
    objs = [os.path.join(OBJ, s[:-4] + '.o') for s in srcs]
    if force or device_jobs or not os.path.exists(LIB) or any(os.path.getmtime(o) > os.path.getmtime(LIB) for o in objs):
        r = subprocess.run([hipcc, '--offload-arch=gfx950', '-shared', '-fPIC', '-o', LIB] + objs, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError('link failed:\n' + r.stderr)
        if verbose:
            print('[build] linked', LIB)
    return LIB


if __name__ == '__main__':
    build(force='--force' in sys.argv)
