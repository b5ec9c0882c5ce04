"""Ahead-of-time build of libn3d.so (HIP, gfx950 only) and of _token_ext.so, the C++ host side of the token operators (against torch's headers).

    python -m next3d_amd.build [--force]

hipcc cross-compiles without a GPU; the resulting in-tree .so travels to the GPU box with the snapshot.
"""
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, 'csrc')
OBJ = os.path.join(HERE, 'build')
LIB = os.path.join(HERE, 'libn3d.so')
EXT = os.path.join(HERE, '_token_ext.so')
HIPCC = os.environ.get('HIPCC', '/opt/rocm/bin/hipcc')
ARCH = 'gfx950'
CFLAGS = ['-O3', '-std=c++17', '-fPIC', f'--offload-arch={ARCH}', '-Wall', '-Wno-unused-function', '-Wno-unused-variable',
          # no packed float32 instructions (v_pk_add / mul / fma_f32), which the optimiser otherwise forms out of ordinary float code: some of their
          # forms have given wrong results on this hardware.  (hipcc's host pass does not know the feature and says so: harmless)
          '-Xclang', '-target-feature', '-Xclang', '-packed-fp32-ops']
# raster.hip mirrors the C oracle operation-for-operation: no FMA contraction there (bit-exact face selection)
PER_FILE = {'raster.hip': ['-ffp-contract=off']}


def _sources():
    return sorted(f for f in os.listdir(CSRC) if f.endswith('.hip'))


def _stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def _other_command(target, cmd):
    """Was `target` built by another command (other flags, another torch)?  Every object has the command that made it beside it."""
    try:
        with open(target + '.cmd') as f:
            return f.read() != ' '.join(cmd)
    except FileNotFoundError:
        return True


def _note_command(target, cmd):
    with open(target + '.cmd', 'w') as f:
        f.write(' '.join(cmd))


def _ext_commands():
    """Compile and link commands of _token_ext.so: host code only, linked against the torch that will load it, whose version is part of them."""
    import sysconfig

    import torch
    root = os.path.dirname(torch.__file__)
    src, obj = os.path.join(CSRC, 'token_ext.cpp'), os.path.join(OBJ, 'token_ext.o')
    includes = [os.path.join(root, 'include'), os.path.join(root, 'include', 'torch', 'csrc', 'api', 'include'), '/opt/rocm/include',
                sysconfig.get_paths()['include']]
    compile_ = ['g++', '-O2', '-std=c++17', '-fPIC', '-Wall', '-D__HIP_PLATFORM_AMD__=1', '-DUSE_ROCM=1', f'-DN3D_TORCH="{torch.__version__}"',
                f'-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}']
    compile_ += [a for i in includes for a in ('-isystem', i)] + ['-c', src, '-o', obj]
    link = ['g++', '-shared', '-fPIC', '-o', EXT, obj, '-L' + os.path.join(root, 'lib'), '-ltorch_python', '-ltorch', '-ltorch_cpu', '-ltorch_hip', '-lc10', '-lc10_hip']
    return src, obj, compile_, link


def build(force=False, verbose=True):
    os.makedirs(OBJ, exist_ok=True)
    headers = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith('.h')]
    headers.append(os.path.join(HERE, '..', 'include', 'n3d.h'))
    jobs = []
    for src in _sources():
        obj = os.path.join(OBJ, src.replace('.hip', '.o'))
        cmd = [HIPCC] + CFLAGS + PER_FILE.get(src, []) + ['-c', os.path.join(CSRC, src), '-o', obj]
        if force or _stale(obj, [os.path.join(CSRC, src)] + headers) or _other_command(obj, cmd):
            jobs.append((obj, cmd))

    ext_src, ext_obj, ext_compile, ext_link = _ext_commands()
    if force or _stale(ext_obj, [ext_src, os.path.join(HERE, '..', 'include', 'n3d.h')]) or _other_command(ext_obj, ext_compile):
        jobs.insert(0, (ext_obj, ext_compile))         # (the longest job first)

    def run(cmd):
        if verbose:
            print('[n3d build]', ' '.join(cmd[-3:]), flush=True)
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f'build failed: {" ".join(cmd)}\n{r.stdout}\n{r.stderr}')
        said = '\n'.join(line for line in r.stderr.splitlines() if 'packed-fp32-ops' not in line)
        if verbose and said.strip():
            print(said, file=sys.stderr)

    def make(job):
        run(job[1])
        _note_command(*job)

    with ThreadPoolExecutor(max_workers=min(8, max(1, len(jobs)))) as ex:
        list(ex.map(make, jobs))
    objs = [os.path.join(OBJ, s.replace('.hip', '.o')) for s in _sources()]
    if force or _stale(LIB, objs):
        run([HIPCC, '-shared', '-fPIC', f'--offload-arch={ARCH}', '-Wl,--no-undefined', '-o', LIB] + objs)
        # a library that links but cannot be loaded (hipcc's host pass silently drops the launch stub of some __global__ templates:
        # an undefined __device_stub__ symbol) must fail HERE, on the build machine, not on the GPU box
        import ctypes
        try:
            import torch                               # noqa: F401  (torch's HIP runtime first: see __graft_entry__.build)
        except ImportError:
            pass
        ctypes.CDLL(LIB)
    if force or _stale(EXT, [ext_obj]):
        run(ext_link)
        subprocess.run([sys.executable, '-c', 'import torch; import importlib.util as u; '
                        f's = u.spec_from_file_location("_token_ext", {EXT!r}); s.loader.exec_module(u.module_from_spec(s))'], check=True)
    return LIB


if __name__ == '__main__':
    print(build(force='--force' in sys.argv))
