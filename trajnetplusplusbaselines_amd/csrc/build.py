"""Build libtrajnet_hip.so (gfx950) in-tree with hipcc.  No torch dependency: the library is a plain
C-ABI shared object (include/trajnet_hip.h); hipcc cross-compiles without a GPU.  Beside it _trajnet_torch.so, host code that
makes autograd nodes of two of its operators."""
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


def needs_build():
    if not (os.path.exists(OUT) and os.path.exists(TORCH_OUT)):
        return True
    t = min(os.path.getmtime(OUT), os.path.getmtime(TORCH_OUT))
    deps = [os.path.join(HERE, f) for f in SOURCES + HEADERS + [TORCH_SOURCE]] + [os.path.abspath(__file__)]
    return any(os.path.exists(d) and os.path.getmtime(d) > t for d in deps)


def torch_command():
    torch = importlib.util.find_spec('torch').submodule_search_locations[0]
    inc = [os.path.join(torch, 'include'), os.path.join(torch, 'include', 'torch', 'csrc', 'api', 'include'), sysconfig.get_paths()['include']]
    return [hipcc(), '-std=c++17', '-O2', '-fPIC', '-shared', '-fvisibility=hidden', '-w'] + ['-I' + i for i in inc] + [
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
    cmds.append(torch_command())
    if verbose:
        print(' '.join(cmds[-1]))
    # translation units are independent: compile them side by side
    from concurrent.futures import ThreadPoolExecutor
    with ThreadPoolExecutor(max_workers=min(len(cmds), os.cpu_count() or 4)) as pool:
        list(pool.map(subprocess.check_call, cmds))
    cmd = [hipcc(), '--offload-arch=gfx950', '-shared', '-fPIC', '-o', OUT] + objs
    if verbose:
        print(' '.join(cmd))
    subprocess.check_call(cmd)
    return OUT


if __name__ == '__main__':
    print(build(force='--force' in sys.argv, verbose=True))
