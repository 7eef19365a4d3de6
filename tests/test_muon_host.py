"""Host-side checks of the operators for matrix-shaped parameters, without a GPU: the library
exports what its header declares, arguments are refused before any device work, the Python surface
refuses what it cannot serve, and what the compiler made of the kernels."""

from __future__ import annotations

import ctypes
import os
import re
import shutil
import subprocess

import pytest
import torch

import torchopt_amd
from conftest import REPO
from torchopt_amd import FusedMuon, MetaMuon, Muon, muon, orthogonalize
from torchopt_amd._C import muon_op
from torchopt_amd.transform import scale_by_muon

HEADER = os.path.join(REPO, 'include', 'toa_muon.h')
LIB = os.path.join(REPO, 'torchopt_amd', 'libtoa_muon.so')
EDTYPE, ENULL, ESIZE, EVALUE, EWORKSPACE = -1, -2, -3, -5, -6
F32, F64, F16, BF16, I8 = 0, 1, 2, 3, 4


class View(ctypes.Structure):
    _fields_ = [('data', ctypes.c_void_p), ('row_stride', ctypes.c_int64),
                ('col_stride', ctypes.c_int64)]


class Series(ctypes.Structure):
    _fields_ = [('steps', ctypes.c_int), ('a', ctypes.c_double), ('b', ctypes.c_double),
                ('c', ctypes.c_double), ('eps', ctypes.c_double)]


class Hyper(ctypes.Structure):
    _fields_ = [('momentum', ctypes.c_double), ('lr', ctypes.c_double),
                ('weight_decay', ctypes.c_double), ('nesterov', ctypes.c_int),
                ('maximize', ctypes.c_int), ('adjust', ctypes.c_int), ('apply', ctypes.c_int)]


@pytest.fixture(scope='module')
def lib():
    lib = ctypes.CDLL(LIB)
    lib.toa_muon_error_string.restype = ctypes.c_char_p
    for name in ('orthogonalize_workspace', 'backward_workspace', 'kept_bytes'):
        getattr(lib, f'toa_muon_{name}').restype = ctypes.c_size_t
    return lib


def sides(*values):
    return (ctypes.c_int64 * len(values))(*values)


def series(steps=5, a=3.4445, b=-4.775, c=2.0315, eps=1e-7):
    return ctypes.byref(Series(steps, a, b, c, eps))


def orth(lib, dtype=F32, rows=(4,), cols=(4,), q=None, data=None, kept=None, kept_size=0,
         workspace=None, size=0):
    views = (View * max(1, len(rows)))(*[View(data, 1, 1) for _ in rows])
    return lib.toa_muon_orthogonalize_multi(
        dtype, ctypes.c_size_t(len(rows)), sides(*rows), sides(*cols), views, views,
        q or series(), ctypes.c_void_p(kept), ctypes.c_size_t(kept_size),
        ctypes.c_void_p(workspace), ctypes.c_size_t(size), None)


def test_library_exports_every_declared_symbol(lib):
    text = re.sub(r'/\*.*?\*/', '', open(HEADER).read(), flags=re.S)
    names = re.findall(r'TOA_API\s+(?:const\s+char\s*\*|int|size_t)\s*(\w+)\s*\(', text)
    assert len(names) == 10
    for name in names:
        assert hasattr(lib, name), f'{name} declared in include/toa_muon.h but not exported'
    assert lib.toa_muon_abi_version() == 1
    for code in (EDTYPE, ENULL, ESIZE, EVALUE, EWORKSPACE):
        assert lib.toa_muon_error_string(code).startswith(b'toa_muon: ')
        assert b'unknown' not in lib.toa_muon_error_string(code)
    assert lib.toa_muon_error_string(0) == b'success'


def test_argument_errors_need_no_device(lib):
    assert orth(lib, rows=(), cols=()) == 0
    assert orth(lib, rows=(0, 3), cols=(5, 0)) == 0  # nothing but empty matrices
    assert orth(lib, dtype=F64) == EDTYPE and orth(lib, dtype=I8) == EDTYPE
    assert orth(lib) == ENULL  # the matrix ...
    assert orth(lib, rows=(100,), cols=(100,), data=256) == ENULL  # ... or the workspace
    need = lib.toa_muon_orthogonalize_workspace(F32, ctypes.c_size_t(1), sides(100), sides(100),
                                                series(), 0, None)
    assert orth(lib, rows=(100,), cols=(100,), data=256, workspace=256, size=need - 1) == EWORKSPACE
    assert orth(lib, rows=(100,), cols=(100,), data=256, workspace=264, size=need) == EWORKSPACE
    keep = lib.toa_muon_kept_bytes(F32, ctypes.c_size_t(1), sides(100), sides(100), series(), None)
    assert keep == 5 * 4 * 128 * 128 * 4  # X, its transpose, S and P of five steps
    for kept, short in ((256, 1), (264, 0)):
        assert orth(lib, rows=(100,), cols=(100,), data=256, kept=kept, kept_size=keep - short,
                    workspace=256, size=need) == EWORKSPACE
    assert orth(lib, rows=((1 << 20) + 1,), cols=(1,)) == ESIZE
    assert orth(lib, rows=(-1,), cols=(4,)) == ESIZE
    inf, nan = float('inf'), float('nan')
    for bad in (dict(steps=0), dict(steps=33), dict(a=nan), dict(b=inf), dict(eps=-1.0),
                dict(eps=nan), dict(a=100.0), dict(c=1e6)):
        assert orth(lib, q=series(**bad)) == EVALUE, bad
        status = ctypes.c_int(0)
        lists = F32, ctypes.c_size_t(1), sides(100), sides(100), series(**bad)
        for size in (lambda: lib.toa_muon_orthogonalize_workspace(*lists, 0, ctypes.byref(status)),
                     lambda: lib.toa_muon_kept_bytes(*lists, ctypes.byref(status))):
            status.value = 0
            assert size() == 0 and status.value == EVALUE, bad
    # the last iterate may grow, as it is not multiplied again
    assert orth(lib, rows=(0,), cols=(0,), q=series(steps=1, a=100.0)) == 0
    assert orth(lib, rows=(0,), cols=(0,), q=series(steps=2, a=100.0)) == EVALUE
    assert lib.toa_muon_orthogonalize_multi(F32, ctypes.c_size_t(0), None, None, None, None, None,
                                            None, ctypes.c_size_t(0), None, ctypes.c_size_t(0),
                                            None) == ENULL


def test_step_arguments(lib):
    def step(dtype=F32, kept=F32, **kw):
        h = dict(momentum=0.95, lr=0.1, weight_decay=0.0, nesterov=1, maximize=0, adjust=1, apply=1)
        h.update(kw)
        return lib.toa_muon_step_multi(dtype, kept, ctypes.c_size_t(0), None, None, None, None,
                                       None, None, ctypes.byref(Hyper(**h)), series(), None,
                                       ctypes.c_size_t(0), None)

    assert step() == 0 and step(BF16, BF16) == 0 and step(BF16, F32) == 0 and step(F16, I8) == 0
    assert step(F32, F16) == EDTYPE and step(F64, F64) == EDTYPE and step(F32, 7) == EDTYPE
    for bad in (dict(momentum=1.0), dict(momentum=-0.1), dict(momentum=float('nan')),
                dict(adjust=3), dict(adjust=-1), dict(lr=float('nan'))):
        assert step(**bad) == EVALUE, bad
    assert step(lr=float('nan'), apply=0) == 0  # read by `apply` only


def test_workspace_sizes(lib):
    def size(rows, cols, steps=5, which='orthogonalize', dtype=F32, keep=0):
        status = ctypes.c_int(99)
        lists = dtype, ctypes.c_size_t(len(rows)), sides(*rows), sides(*cols), series(steps)
        if which == 'kept':
            return lib.toa_muon_kept_bytes(*lists, ctypes.byref(status)), status.value
        n = getattr(lib, f'toa_muon_{which}_workspace')(*lists, keep, ctypes.byref(status))
        return n, status.value

    assert size((), ()) == (0, 0) and size((0,), (7,)) == (0, 0)
    assert size((32,), (288,)) == (0, 0)  # small: registers and LDS, no workspace
    assert size((1024,), (1024,))[0] == size((1024,), (1024,), dtype=BF16)[0]
    assert size((100,), (300,)) == size((300,), (100,))
    # one batch holds at most 4 GiB of regions, whatever the list
    assert size((1024,) * 400, (1024,) * 400)[0] < (4 << 30) + (64 << 20)
    assert size((1024,), (1024,), which='backward')[0] > 3 * size((1024,), (1024,))[0]
    # what is kept is not in the workspace; small matrices keep nothing
    kept = size((1024,), (1024,), which='kept')[0]
    whole, rest = (size((1024,), (1024,), which='backward', keep=k)[0] for k in (0, 1))
    assert whole - rest == kept == 5 * 4 * 4 << 20
    assert size((32, 1024), (288, 1024), which='kept')[0] > kept  # (they go along with a larger one)
    assert size((32,), (288,), which='kept') == (0, 0)
    # (in a long series the way back measures its norms, which the small form does not)
    assert size((32,), (288,), which='kept', steps=8)[0] > 0
    assert size((1024,), (1024,), keep=1)[0] < size((1024,), (1024,))[0]
    assert size((4,), (4,), steps=0)[1] == EVALUE and size((4,), (4,), dtype=F64)[1] == EDTYPE
    assert size((1 << 21,), (4,))[1] == ESIZE


def test_block_lists_without_device(lib):
    assert lib.toa_muon_quantize_multi(F64, ctypes.c_size_t(0), None, None, None, None, None) == EDTYPE
    assert lib.toa_muon_quantize_multi(F32, ctypes.c_size_t(0), None, None, None, None, None) == 0
    n = (ctypes.c_size_t * 1)(5)
    assert lib.toa_muon_quantize_multi(F32, ctypes.c_size_t(1), None, n, None, None, None) == ENULL
    zero = (ctypes.c_size_t * 1)(0)
    assert lib.toa_muon_dequantize_multi(F32, ctypes.c_size_t(1), None, None, zero, None, None) == 0


def test_cpu_and_meta_tensors_are_refused_not_computed():
    for device in ('cpu', 'meta'):
        x = torch.ones(4, 4, device=device)
        for fn, args in [
            (muon_op.orthogonalize_multi, ([x],)),
            (muon_op.orthogonalize_backward_multi, ([x], [x])),
            (muon_op.forward_multi_, ([x], [x.clone()], None, 0.9)),
            (muon_op.fused_step_multi_, ([x], [x.clone()], [x.clone()], None, 0.9, 0.1)),
            (muon_op.quantize_multi, ([x],)),
            (muon_op.dequantize_multi_, ([x], [x.to(torch.int8)], [x])),
            (orthogonalize, (x,)), (torchopt_amd.quantize_blocks, (x,)),
        ]:
            with pytest.raises(RuntimeError, match='Not implemented'):
                fn(*args)


def test_empty_lists_and_types():
    assert muon_op.orthogonalize_multi([]) == [] and orthogonalize([]) == [] and orthogonalize(()) == ()
    assert muon_op.quantize_multi([]) == ([], [])
    assert torchopt_amd.quantize_blocks([]) == ([], [])
    assert torchopt_amd.dequantize_blocks([], []) == []
    with pytest.raises(TypeError):
        orthogonalize([1.0])
    with pytest.raises(TypeError):
        muon_op.orthogonalize_multi([1.0])
    with pytest.raises(ValueError):
        muon_op.forward_multi_([], [], None, 0.9, adjust_lr_fn='unheard of')


def test_optimizer_arguments():
    p = [torch.ones(3, 4)]
    for kwargs in (dict(lr=-1.0), dict(weight_decay=-0.1), dict(momentum=1.0), dict(momentum=-0.1),
                   dict(ns_steps=0), dict(ns_steps=33), dict(eps=-1e-7),
                   dict(ns_coefficients=(1.0, 2.0)), dict(ns_coefficients=(1.0, 2.0, float('inf'))),
                   dict(adjust_lr_fn='unheard of'), dict(momentum_dtype=torch.float16)):
        with pytest.raises(ValueError):
            FusedMuon(p, **kwargs)
    for kwargs in (dict(momentum=1.0), dict(ns_steps=0), dict(adjust_lr_fn='x')):
        with pytest.raises(ValueError):
            scale_by_muon(**kwargs)
        with pytest.raises(ValueError):
            muon(**kwargs)
    with pytest.raises(TypeError):
        FusedMuon([1.0])
    for bad in (torch.ones(3), torch.ones(()), torch.ones(3, 4, dtype=torch.float64)):
        with pytest.raises(ValueError):
            FusedMuon([bad])
        with pytest.raises(ValueError):
            scale_by_muon().init([bad])
    with pytest.raises(RuntimeError):
        MetaMuon([torch.ones(3, 3)])
    assert Muon is FusedMuon


def test_optimizer_state_before_and_after_init():
    p = [torch.ones(3, 4), torch.ones(2, 3, 5).to(memory_format=torch.contiguous_format)]
    opt = FusedMuon(p, momentum_dtype=torch.int8)
    assert opt.state_dict() == (None,)
    assert opt.step() is None  # no gradients: nothing is launched
    opt.zero_grad()
    (taken, state), = opt.state_dict()
    assert taken == 0 and [m.dtype for m in state.momentum] == [torch.int8] * 2
    assert [s.numel() for s in state.scales] == [1, 1]
    opt.load_state_dict(opt.state_dict())
    opt.load_state_dict((None,))
    for bad in ((), (None, None), ((0, state._replace(momentum=state.momentum[:1])),),
                ((0, state._replace(momentum=state.momentum[::-1])),)):
        with pytest.raises(ValueError):
            opt.load_state_dict(bad)
    p[0].grad = torch.ones(3, 4)
    with pytest.raises(RuntimeError, match='Not implemented'):  # CPU parameters are refused
        opt.step()


def test_functional_state_and_partition():
    t = {'w': torch.ones(3, 4), 'b': torch.ones(4), 'none': None}
    state = muon().init(t)
    part = state[1]
    assert part.keys == ('w', 'b', 'none')
    assert part.matrices.momentum[0].shape == (3, 4) and part.matrices.momentum[1:] == [None, None]
    assert part.others.mu[0] is None and part.others.mu[1].shape == (4,)
    only = scale_by_muon(momentum_dtype=torch.int8)
    s = only.init([t['w'], None])
    assert s.momentum[0].dtype == torch.int8 and s.momentum[1] is None and s.scales[1] is None
    # nothing to do: no gradient, or no state
    out, s2 = only.update([None, None], s)
    assert out == [None, None] and s2.momentum[0] is s.momentum[0]
    with pytest.raises(ValueError, match='different tree structures'):
        only.update([None], s)
    with pytest.raises(ValueError, match='in place only'):
        only.update([t['w'], None], s, inplace=False)


# ---- what the compiler made of the kernels -------------------------------------------------

LLVM = '/opt/rocm/llvm/bin'


@pytest.fixture(scope='module')
def code_object(tmp_path_factory):
    tools = [os.path.join(LLVM, t) for t in ('llvm-objcopy', 'clang-offload-bundler', 'llvm-objdump',
                                             'llvm-readelf')]
    if not all(os.path.exists(t) for t in tools) or not os.path.exists(LIB):
        pytest.skip('needs the built library and the LLVM tools of ROCm')
    tmp = tmp_path_factory.mktemp('muon_code_object')
    fatbin, code = str(tmp / 'fatbin'), str(tmp / 'gfx950.co')
    subprocess.run([tools[0], '--dump-section', f'.hip_fatbin={fatbin}', LIB, os.devnull], check=True)
    subprocess.run([tools[1], '--unbundle', '--type=o', f'--input={fatbin}',
                    '--targets=hipv4-amdgcn-amd-amdhsa--gfx950', f'--output={code}'], check=True)
    return code


def _registers(operand):
    m = re.match(r'v\[(\d+):(\d+)\]$', operand) or re.match(r'v(\d+)()$', operand)
    if not m:
        return set()
    return set(range(int(m[1]), int(m[2] or m[1]) + 1))


def test_nothing_writes_an_operand_right_behind_its_matrix_instruction(code_object):
    """A write into a register that the matrix instruction just before reads has been lost on this
    hardware (muon_kernels.hpp, beforeMatrix): no kernel may hold one as the next vector
    instruction, unless idle cycles stand between.  And no packed float32 arithmetic, as in the
    other library."""
    text = subprocess.run([os.path.join(LLVM, 'llvm-objdump'), '-d', '--no-show-raw-insn',
                           code_object], check=True, capture_output=True, text=True).stdout
    for banned in ('v_pk_add_f32', 'v_pk_mul_f32', 'v_pk_fma_f32'):
        assert banned not in text, banned
    seen, recent, bad = 0, [], []
    for line in text.splitlines():
        words = line.split('//')[0].replace(',', ' ').split()
        if not words or words[0].endswith(':') or line[:1] != '\t':
            recent = []
            continue
        op = words[0]
        if op.startswith('v_mfma'):
            seen += 1
            recent = [(line, _registers(words[2]) | _registers(words[3]))]
            continue
        if op == 's_nop':  # so many more slots
            recent = recent if int(words[1], 0) == 0 else []
            continue
        if op.startswith('v_') and len(words) > 1:
            written = _registers(words[1])
            bad += [(m.strip(), line.strip()) for m, regs in recent if written & regs]
        recent = [(m, regs) for m, regs in recent] if len(recent) and not op.startswith('v_') else []
    assert seen > 1000
    assert not bad, bad[:3]


def test_the_product_kernels_neither_spill_nor_outgrow_lds(code_object):
    notes = subprocess.run([os.path.join(LLVM, 'llvm-readelf'), '--notes', code_object], check=True,
                           capture_output=True, text=True).stdout
    found, current = {}, None
    for line in notes.splitlines():
        m = re.match(r'(  - |    )\.(\w+):\s*(\S*)\s*$', line)
        if not m:
            continue
        if m[1] == '  - ':
            current = {}
        if current is None:
            continue
        if m[2] == 'name':
            found[m[3]] = current
        elif m[3].lstrip('-').isdigit():
            current[m[2]] = int(m[3])
    product = {n: k for n, k in found.items() if 'gemm_kernel' in n}
    assert len(product) >= 24 and len(found) > 70
    for name, k in found.items():
        assert k['wavefront_size'] == 64 and k['group_segment_fixed_size'] <= 160 << 10, name
        if 'small_kernel' not in name:  # (two rows of blocks: a few spilled registers there)
            assert k['vgpr_spill_count'] == 0 and k['private_segment_fixed_size'] == 0, name
    if shutil.which('c++filt') is None:
        pytest.skip('names as the compiler spells them only')
