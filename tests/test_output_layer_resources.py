"""The tile kernels keep 256 x 256 accumulators in all of a wave's AGPRs, with
hand-counted waits for the DMA in flight: a spill is scratch traffic that those
counts do not know.  None of the kernels as built may have one."""
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LLVM = '/opt/rocm/llvm/bin'


@pytest.mark.parametrize('source,kernels', [
    ('class_logits', ['class_tile_kernel', 'pack_rows_kernel',
                      'part_max_kernel', 'part_stats_kernel',
                      'join_stats_kernel', 'sum_rows_kernel']),
    ('int8_linear', ['int8_tile_kernel', 'quantize_rows_kernel',
                     'dequantize_rows_kernel'])])
def test_no_vector_spills(source, kernels, tmp_path):
    import __graft_entry__ as g
    g.build()
    obj = os.path.join(ROOT, 'build', 'obj', source + '.hip.o')
    if not os.path.exists(obj) or not os.path.isdir(LLVM):
        pytest.skip('no object files of the build')
    bundle, code = str(tmp_path / 'bundle'), str(tmp_path / 'code')
    subprocess.check_call([os.path.join(LLVM, 'llvm-objcopy'),
                           '--dump-section', '.hip_fatbin=' + bundle, obj,
                           str(tmp_path / 'copy.o')])
    subprocess.check_call([os.path.join(LLVM, 'clang-offload-bundler'),
                           '--unbundle', '--type=o', '--input=' + bundle,
                           '--targets=hipv4-amdgcn-amd-amdhsa--gfx950',
                           '--output=' + code])
    notes = subprocess.check_output(
        [os.path.join(LLVM, 'llvm-readelf'), '--notes', code],
        universal_newlines=True)
    seen = set()
    name = None
    for line in notes.splitlines():
        m = re.match(r'\s+\.(name|private_segment_fixed_size|'
                     r'vgpr_spill_count):\s+(\S+)', line)
        if not m:
            continue
        if m.group(1) == 'name':
            if m.group(2).startswith('_Z'):
                name = m.group(2)
                seen.update(k for k in kernels if k in name)
        elif name:
            assert m.group(2) == '0', (name, line)
    assert seen == set(kernels)
