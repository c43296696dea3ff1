"""Build libtrajnet_hip.so (gfx950) in-tree with hipcc.  No torch dependency: the library is a plain
C-ABI shared object (include/trajnet_hip.h); hipcc cross-compiles without a GPU.

Beside it, where a torch for ROCm is installed, _trajnet_torch.so: host code that makes autograd nodes of two of the library's operators
(vocab.py).  The library is linked first and does not depend on it."""
import importlib.util
import os
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
PKG = os.path.dirname(HERE)
OUT_DIR = os.path.join(PKG, 'lib')
OUT = os.path.join(OUT_DIR, 'libtrajnet_hip.so')
TORCH_OUT = os.path.join(OUT_DIR, '_trajnet_torch.so')     # autograd nodes in C++: links against torch, not against OUT
TORCH_SOURCE = 'vocab_torch.cpp'
SOURCES = ['gemm_f32_mfma.hip', 'gemm_skinny.hip', 'gemm_wgrad.hip', 'pool_grid.hip', 'pool_embed_sparse.hip', 'pool_nongrid.hip', 'lstm_seq.hip', 'lstm_bwd.hip', 'loss.hip',
           'optim.hip', 'classical.hip', 'token_embed.hip', 'vocab_ce.hip', 'ndjson_io.cpp']
EXACT = ('classical.hip', 'pool_grid.hip', 'optim.hip')
# units compiled without v_pk_{add,mul,fma}_f32
NO_PACKED_FP32 = ('token_embed.hip', 'vocab_ce.hip')
HEADERS = ['tnp_internal.h', 'vocab_types.h', 'vocab_gemm.h', 'lstm_cell.h', 'classical_core.h', 'grid_build_body.h', os.path.join('..', '..', 'include', 'trajnet_hip.h'),
           os.path.join('..', '..', 'include', 'trajnet_hip_profile.h')]
FLAGS = ['--offload-arch=gfx950', '-O3', '-std=c++17', '-fPIC', '-fno-fast-math', '-fvisibility=hidden',
         '-Wall', '-Wno-unused-function']


def hipcc():
    for c in (os.environ.get('HIPCC'), '/opt/rocm/bin/hipcc', 'hipcc'):
        if c and (os.path.isabs(c) and os.path.exists(c) or not os.path.isabs(c)):
            return c
    return 'hipcc'


def torch_folder():
    """folder of an installed torch for ROCm, or None"""
    spec = importlib.util.find_spec('torch')
    folder = spec.submodule_search_locations[0] if spec and spec.submodule_search_locations else None
    return folder if folder and os.path.exists(os.path.join(folder, 'lib', 'libc10_hip.so')) else None


def needs_build():
    outs = [OUT] + ([TORCH_OUT] if torch_folder() else [])
    if not all(os.path.exists(o) for o in outs):
        return True
    t = min(os.path.getmtime(o) for o in outs)
    deps = [os.path.join(HERE, f) for f in SOURCES + HEADERS + [TORCH_SOURCE]] + [os.path.abspath(__file__)]
    return any(os.path.exists(d) and os.path.getmtime(d) > t for d in deps)


def torch_command():
    """None where there is no torch for ROCm"""
    torch = torch_folder()
    if torch is None:
        return None
    inc = [os.path.join(torch, 'include'), os.path.join(torch, 'include', 'torch', 'csrc', 'api', 'include'), sysconfig.get_paths()['include']]
    # warnings of this file, not of torch's headers
    return [hipcc(), '-std=c++17', '-O2', '-fPIC', '-shared', '-fvisibility=hidden', '-Wall'] + [a for i in inc for a in ('-isystem', i)] + [
        os.path.join(HERE, TORCH_SOURCE), '-o', TORCH_OUT, '-L' + os.path.join(torch, 'lib'), '-ltorch_python', '-ltorch_cpu', '-lc10', '-lc10_hip']


def build(force=False, verbose=False):
    if not (force or needs_build()):
        return OUT
    os.makedirs(OUT_DIR, exist_ok=True)
    objs, cmds = [], []
    for src in SOURCES:
        path = os.path.join(HERE, src)
        if not os.path.exists(path):
            continue
        obj = os.path.join(OUT_DIR, os.path.splitext(src)[0] + '.o')
        # exact-arithmetic units (cell indexing, float64 / float32 simulators): no fma contraction
        extra = ['-ffp-contract=off'] if src in EXACT else []
        if src in NO_PACKED_FP32:
            extra = extra + ['-Xclang', '-target-feature', '-Xclang', '-packed-fp32-ops']
        cmd = [hipcc()] + FLAGS + extra + os.environ.get('TNP_HIPCC_EXTRA', '').split() + ['-c', path, '-o', obj]
        if verbose:
            print(' '.join(cmd))
        cmds.append(cmd)
        objs.append(obj)
    torch_cmd = torch_command()
    if verbose:
        print(' '.join(torch_cmd) if torch_cmd else 'no torch for ROCm: %s is not built' % TORCH_OUT)
    # translation units are independent: compile them side by side
    from concurrent.futures import ThreadPoolExecutor
    with ThreadPoolExecutor(max_workers=min(len(cmds) + 1, os.cpu_count() or 4)) as pool:
        beside = pool.submit(subprocess.check_call, torch_cmd) if torch_cmd else None
        list(pool.map(subprocess.check_call, cmds))
        cmd = [hipcc(), '--offload-arch=gfx950', '-shared', '-fPIC', '-o', OUT] + objs
        if verbose:
            print(' '.join(cmd))
        subprocess.check_call(cmd)
    if beside:
        beside.result()                  # raises what the torch file's compiler said, the library being there
    return OUT


if __name__ == '__main__':
    print(build(force='--force' in sys.argv, verbose=True))
