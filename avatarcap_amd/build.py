"""In-tree build of libavcap_hip.so for gfx950 with hipcc (cross-compiles without a GPU).

`python -m avatarcap_amd.build` or `__graft_entry__.build()`.  The .so stays in the package
directory so it travels with the repository snapshot to the GPU box.
"""
from __future__ import annotations

import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, 'csrc')
OBJ = os.path.join(HERE, 'csrc', '_obj')
LIB = os.path.join(HERE, 'libavcap_hip.so')
SOURCES = ['fused_mlp.hip', 'conv_enc.hip', 'misc.hip', 'mesh.hip', 'raster.hip', 'fusion.hip', 'knn_lbs.hip', 'render.hip', 'linear.hip', 'layer_norm.hip', 'pack.cpp', 'capi.cpp']
HEADERS = ['avcap_internal.h', 'linear.h', 'mlp_layout.h', 'mc_tables.h', 'store_settle.h', os.path.join('..', '..', 'include', 'avcap.h')]
HIPCC = os.environ.get('HIPCC', '/opt/rocm/bin/hipcc')
FLAGS = ['--offload-arch=gfx950', '-O3', '-std=c++17', '-fPIC', '-Wno-unused-value', '-Wno-unused-result']
# gfx950 / ROCm 7.2: a VGPR written by a packed-f32 VALU instruction and read as the data of a multi-dword store an instruction later reached memory stale in
# the wave's last 16 lanes when another kernel shared the CU (csrc/store_settle.h, profiles/r06_store_hazard.md).  hipcc forms those instructions by itself
# (SLP-packing of adjacent scalar f32 operations); the element-wise translation units are built without them -- same IEEE operations, one per instruction --,
# the two MFMA units (fused_mlp.hip: no packed producer near any wide store; conv_enc.hip: its element-wise kernels settle() their stores) keep their code.
NOPK = ['-Xclang', '-target-feature', '-Xclang', '-packed-fp32-ops']
# mesh / KNN kernels promise bit-exact agreement with the C oracle (built with -ffp-contract=off):
# HIP's __fmul_rn/__fadd_rn are plain operators, so contraction has to be disabled per file.
EXTRA = {'mesh.hip': ['-ffp-contract=off'] + NOPK, 'knn_lbs.hip': ['-ffp-contract=off'] + NOPK, 'raster.hip': ['-ffp-contract=off'] + NOPK, 'render.hip': ['-ffp-contract=off'] + NOPK,
         'misc.hip': NOPK, 'fusion.hip': NOPK, 'linear.hip': NOPK, 'layer_norm.hip': NOPK, 'linear_tile.hip': NOPK,
         # MFMA accumulators in VGPRs: the epilogue reads them without a v_accvgpr_read per value (-0.7 % launch time, tools/ablate_run.sh)
         # (fused_mlp.hip without packed f32 as well: hipcc's SLP-packed v_pk_*_f32 cost issue time beside the MFMAs -- same-box A/B of the dense launch -1.0 % shader cycles)
         # -amdgpu-sched-strategy=max-ilp: what the scheduler does with the code between the pinned pieces; same bits, -1.1 % shader cycles per dense launch (tools/ab_flags.sh;
         # max-memory-clause -0.4 %, no post-RA scheduler +2 %, -O2 the same)
         'fused_mlp.hip': ['-mllvm', '-amdgpu-mfma-vgpr-form', '-mllvm', '-amdgpu-sched-strategy=max-ilp'] + NOPK}


ASAN_PLAIN = {'fused_mlp.hip'}      # translation units left uninstrumented in the --asan flavour (see build())


def _stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def build(force: bool = False, verbose: bool = True, asan: bool = False) -> str:
    """asan=True: the AddressSanitizer flavour (host AND device code instrumented: -fsanitize=address -shared-libasan, gfx950:xnack+) as
    libavcap_hip_asan.so next to the product library -- tools/sanitize/run_asan.sh runs the ragged-size GPU tests against it."""
    global OBJ, LIB, FLAGS
    if asan:
        OBJ, LIB = os.path.join(HERE, 'csrc', '_obj_asan'), os.path.join(HERE, 'libavcap_hip_asan.so')
        FLAGS = ['--offload-arch=gfx950:xnack+', '-O1', '-fsanitize=address', '-shared-libasan', '-std=c++17', '-fPIC', '-Wno-unused-value', '-Wno-unused-result']
    os.makedirs(OBJ, exist_ok=True)
    hdrs = [os.path.join(CSRC, h) for h in HEADERS]
    jobs = []
    # (object name, source, extra flags): fused_mlp.hip is built twice -- the plain kernels and the range-checking flavour
    # (include/avcap.h avc_set_range_check), which live in different namespaces of the same library
    # and a third time with the Softplus layers' weight scale undone in the epilogue (-DAVC_LAYER_SCALE=1: namespace `scaled`, pack.cpp add_warp)
    units = [(src + '.o', src, []) for src in SOURCES] + [('fused_mlp_checked.o', 'fused_mlp.hip', ['-DAVC_CHECK_RANGE=1']),
                                                          ('fused_mlp_scaled.o', 'fused_mlp.hip', ['-DAVC_LAYER_SCALE=1'])]
    # the dense layer's tiled products, once per element type
    units += [(f'linear_tile_{t}.o', 'linear_tile.hip', [f'-DAVC_LIN_{t.upper()}=1']) for t in ('f32', 'bf16', 'f16')]
    for obj, src, extra in units:
        sp = os.path.join(CSRC, src)
        op = os.path.join(OBJ, obj)
        if force or _stale(op, [sp] + hdrs):
            flags = FLAGS
            if asan and src in ASAN_PLAIN:             # hipcc 7.2 crashes instrumenting these hand-scheduled kernels: built plain (same xnack+ target) into the ASAN library
                flags = ['--offload-arch=gfx950:xnack+', '-O3', '-std=c++17', '-fPIC', '-Wno-unused-value', '-Wno-unused-result']
            cmd = [HIPCC] + flags + EXTRA.get(src, []) + extra + (['-x', 'hip'] if src.endswith('.cpp') else []) + ['-c', sp, '-o', op]
            jobs.append((obj, cmd))

    def run(job):
        src, cmd = job
        if verbose:
            print('[avatarcap_amd.build]', ' '.join(cmd), flush=True)
        subprocess.check_call(cmd)

    with ThreadPoolExecutor(max_workers=4) as ex:
        list(ex.map(run, jobs))
    objs = [os.path.join(OBJ, u[0]) for u in units]
    if force or jobs or _stale(LIB, objs):
        cmd = [HIPCC, '--offload-arch=gfx950:xnack+' if asan else '--offload-arch=gfx950', '-shared', '-fPIC'] + (['-fsanitize=address', '-shared-libasan'] if asan else []) + objs + ['-o', LIB]
        if verbose:
            print('[avatarcap_amd.build]', ' '.join(cmd), flush=True)
        subprocess.check_call(cmd)
    return LIB


if __name__ == '__main__':
    build(force='--force' in sys.argv, asan='--asan' in sys.argv)
