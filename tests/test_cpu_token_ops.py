"""CPU tests of the token operators: what they refuse, before anything reaches a device."""
import ctypes as C
import os
import subprocess

import pytest
import torch

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _raises(match, fn, *args, **kw):
    with pytest.raises(RuntimeError, match=match):
        fn(*args, **kw)


def test_layer_norm_refusals():
    from next3d_amd.torch_utils.ops.layer_norm import layer_norm
    x = torch.zeros(3, 8)
    _raises('HIP device only', layer_norm, x)
    _raises('must be', layer_norm, x.double())
    _raises('must be', layer_norm, x.long())
    _raises('tensor', layer_norm, [1.0])
    _raises('last dimension', layer_norm, torch.zeros(()))
    _raises('last dimension', layer_norm, torch.zeros(3, 0))
    _raises('7 elements for 8', layer_norm, x, torch.ones(7))
    _raises('dimensions', layer_norm, x, torch.ones(1, 8))
    _raises('weight must be', layer_norm, x, torch.ones(8).half())
    _raises('bias must be', layer_norm, x.half(), None, torch.ones(8).bfloat16())
    _raises('one dtype', layer_norm, x.half(), torch.ones(8).half(), torch.ones(8))
    for eps in (-1e-6, float('nan'), float('inf')):
        _raises('eps', layer_norm, x, eps=eps)


def test_rotary_refusals():
    from next3d_amd.torch_utils.ops.rotary import rotary
    q, pos = torch.zeros(2, 5, 3, 16), torch.zeros(5, 2, dtype=torch.int32)
    _raises('HIP device only', rotary, q, pos, (8, 8))
    _raises('4 dimensions', rotary, q[0], pos, (8, 8))
    _raises('q must be', rotary, q.double(), pos, (8, 8))
    _raises('k must be', rotary, q, pos, (8, 8), k=q.half())
    _raises('does not have', rotary, q, pos, (8, 8), k=q[:, :4])
    _raises('does not have', rotary, q, pos, (8, 8), k=q[..., :8])
    _raises('positions must be', rotary, q, pos.short(), (8, 8))
    _raises('positions must be', rotary, q, pos[:4], (8, 8))
    _raises('positions must be', rotary, q, pos, (4, 4, 8))
    _raises('positions must be', rotary, q, pos[None].expand(3, 5, 2), (8, 8))
    for sections in ((), (3, 5), (8, 16), (-2, 8), (0, 0), (2, 2, 2, 2, 2)):
        _raises('sections', rotary, q, pos, sections)
    _raises('pairing', rotary, q, pos, (8, 8), pairing='quarters')
    _raises('ladder', rotary, q, pos, (8, 8), ladder='rope')
    for base in (0.0, -1.0, float('inf'), float('nan')):
        _raises('base', rotary, q, pos, (8, 8), base=base)
    _raises('no gradient', rotary, q, pos.float().requires_grad_(), (8, 8))
    _raises('channels', rotary, torch.zeros(1, 5, 1, 1026), pos, (8, 8))
    _raises('heads', rotary, torch.zeros(1, 5, 4097, 16), pos, (8, 8))


def _struct_layout(tmp_path, cname, cls):
    lines = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{os.path.join(REPO, "include", "n3d.h")}"', 'int main(void) {', f'  printf("size %zu\\n", sizeof({cname}));']
    lines += [f'  printf("{name} %zu\\n", offsetof({cname}, {name}));' for name, _ in cls._fields_] + ['  return 0;', '}']
    src, exe = tmp_path / 'layout.c', tmp_path / 'layout'
    src.write_text('\n'.join(lines))
    subprocess.run(['gcc', '-std=c11', str(src), '-o', str(exe)], check=True)
    out = dict(line.split() for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines())
    assert int(out.pop('size')) == C.sizeof(cls)
    assert {k: int(v) for k, v in out.items()} == {name: getattr(cls, name).offset for name, _ in cls._fields_}


def test_rotary_descriptor_layout(tmp_path):
    from next3d_amd import _lib
    _struct_layout(tmp_path, 'n3d_rotary_desc', _lib.RotaryDesc)


def test_c_entries_refuse_bad_calls():
    """The library's own checks (a C caller has no Python in front of it): they return before any launch, so they hold without a device."""
    from next3d_amd import _lib
    lib = _lib.lib()

    def err(rc):
        assert rc != 0
        return lib.n3d_last_error().decode()

    p = 4096                                                       # never dereferenced: every call below is refused
    assert 'dtype' in err(lib.n3d_layer_norm(p, None, None, p, None, None, 1, 8, 8, 7, 0, 1e-5, None))
    assert 'sizes' in err(lib.n3d_layer_norm(p, None, None, p, None, None, 1, 0, 8, 0, 0, 1e-5, None))
    assert 'null' in err(lib.n3d_layer_norm(None, None, None, p, None, None, 1, 8, 8, 0, 0, 1e-5, None))
    assert 'null' in err(lib.n3d_layer_norm(p, None, None, p, p, None, 1, 8, 8, 0, 0, 1e-5, None))
    assert 'weight' in err(lib.n3d_layer_norm(p, p, None, p, None, None, 1, 8, 8, 1, 2, 1e-5, None))
    assert 'eps' in err(lib.n3d_layer_norm(p, p, None, p, None, None, 1, 8, 8, 1, 1, -1.0, None))
    assert lib.n3d_layer_norm(None, None, None, None, None, None, 0, 8, 8, 0, 0, 1e-5, None) == 0
    assert 'rows' in err(lib.n3d_layer_norm_bwd(p, p, None, p, p, p, None, None, None, 0, 8, 8, 8, 0, 0, None))
    assert 'null' in err(lib.n3d_layer_norm_bwd(p, p, None, p, p, p, p, None, None, 1, 8, 8, 8, 0, 0, None))
    assert lib.n3d_layer_norm_bwd_workspace(0, 8, 0) == 0

    def rot(**kw):
        d = _lib.RotaryDesc(q=p, positions=p, out_q=p, pos_token_stride=1, base=1e4, B=1, L=2, heads_q=1, D=16, axes=1, dtype=0)
        d.sections[0] = 16
        for k, v in kw.items():
            if k == 'sections':
                d.sections[:] = v
            else:
                setattr(d, k, v)
        return lib.n3d_rotary(d, None)

    for kw, word in ((dict(axes=5), 'axes'), (dict(axes=0), 'axes'), (dict(D=1), 'channels'), (dict(D=2048), 'channels'), (dict(dtype=4), 'dtype'),
                     (dict(pos_type=3), 'positions'), (dict(positions=None), 'positions'), (dict(base=0.0), 'base'), (dict(q=None), 'null'),
                     (dict(heads_k=1), 'null'), (dict(sections=(3, 0, 0, 0)), 'even'), (dict(sections=(18, 0, 0, 0)), 'even'), (dict(sections=(0, 0, 0, 0)), 'add up'),
                     (dict(axes=2, sections=(16, 16, 0, 0)), 'add up'), (dict(L=-1), 'negative'),
                     (dict(B=2 ** 16, L=2 ** 16), 'tokens')):
        assert word in err(rot(**kw)), kw
    assert rot(L=0) == 0
    assert 'null' in err(lib.n3d_rotary(None, None))


def test_attention_refusals():
    from next3d_amd.torch_utils.ops.attention import attention
    q, k = torch.zeros(2, 5, 4, 16).half(), torch.zeros(2, 7, 2, 16).half()
    i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32)
    _raises('HIP device only', attention, q, k, k)
    _raises('4 dimensions', attention, q[0], k, k)
    _raises('q must be', attention, q.float(), k, k)
    _raises('k must be', attention, q, k.bfloat16(), k)
    _raises('v must be', attention, q, k, k.float())
    _raises('do not match', attention, q, k, k[:, :6])
    _raises('do not match', attention, q, k[:1], k[:1])
    _raises('do not match', attention, q[..., :8], k, k)
    _raises('multiple of', attention, q[:, :, :3], k, k)
    _raises('multiple of', attention, q, k[:, :, :0], k[:, :, :0])
    _raises('head sizes', attention, q[..., :12], k[..., :12], k[..., :12])
    _raises('head sizes', attention, torch.zeros(1, 2, 1, 136).half(), torch.zeros(1, 2, 1, 136).half(), torch.zeros(1, 2, 1, 136).half())
    for kw in (dict(scale=float('nan')), dict(scale=float('inf')), dict(softcap=-1.0), dict(softcap=float('inf'))):
        _raises('finite', attention, q, k, k, **kw)
    _raises('causal', attention, q, k, k, prefix=i32(2))
    _raises('prefix must be', attention, q, k, k, prefix=i32(3), causal=True)
    _raises('prefix must be', attention, q, k, k, prefix=i32(2).long(), causal=True)
    _raises('lengths must', attention, q, k, k, lengths=i32(2, 1))
    _raises('key_documents', attention, q, k, k, documents=i32(2, 5))
    _raises('documents must be', attention, q, k, k, documents=i32(2, 7), key_documents=i32(2, 7))
    _raises('key_documents must be', attention, q, k, k, documents=i32(2, 5), key_documents=i32(2, 5))
    _raises('need documents', attention, q, k, k, key_documents=i32(2, 7))
    _raises('slopes for', attention, q, k, k, slopes=torch.zeros(2))
    _raises('slopes must', attention, q, k, k, slopes=torch.zeros(4).half())
    _raises('no gradient', attention, q, k, k, slopes=torch.zeros(4, requires_grad=True))


def test_attention_descriptor_layout(tmp_path):
    from next3d_amd import _lib
    _struct_layout(tmp_path, 'n3d_attention_desc', _lib.AttentionDesc)


def test_attention_c_entries_refuse_bad_calls():
    from next3d_amd import _lib
    lib = _lib.lib()

    def desc(**kw):
        p = 4096                                                   # never dereferenced: every call below is refused
        d = _lib.AttentionDesc(q=p, k=p, v=p, out=p, lse=p, dout=p, dq=p, dk=p, dv=p, scale=1.0, B=1, Lq=4, Lk=300, heads_q=2, heads_k=1, D=16, dtype=1)
        for name, value in dict(dict(q_strides=(128, 32, 16), k_strides=(4800, 16, 16), v_strides=(4800, 16, 16), dout_strides=(128, 32, 16)), **kw).items():
            if name.endswith('_strides'):
                getattr(d, name)[:] = value
            else:
                setattr(d, name, value)
        return d

    shared = ((dict(dtype=0), 'float16'), (dict(D=12), 'head sizes'), (dict(D=136), 'head sizes'), (dict(heads_q=3, heads_k=2), 'multiple'), (dict(heads_k=0), 'multiple'),
              (dict(B=-1), 'negative'), (dict(softcap=-1.0), 'softcap'), (dict(scale=float('nan')), 'scale'), (dict(prefix=4096), 'causal'), (dict(q_documents=4096), 'documents'),
              (dict(q=None), 'null'), (dict(v=None), 'null'), (dict(k_strides=(4800, 15, 16)), 'strides'), (dict(v_strides=(4800, 1 << 24, 16)), 'strides'),
              (dict(q_strides=(128, 32, -16)), 'strides'), (dict(k=4100), 'aligned'), (dict(B=1 << 20, Lq=1 << 14), 'rows'))
    for entry, size in ((lib.n3d_attention, lib.n3d_attention_workspace), (lib.n3d_attention_bwd, lib.n3d_attention_bwd_workspace)):
        for kw, word in shared:
            assert entry(desc(**kw), None) != 0 and word in lib.n3d_last_error().decode(), (kw, lib.n3d_last_error())
            assert size(desc(**kw)) == -1 and word in lib.n3d_last_error().decode(), kw
        need = size(desc())
        assert need > 0
        for kw in (dict(), dict(workspace=4096, workspace_bytes=need - 1), dict(workspace=4104, workspace_bytes=need)):
            assert entry(desc(**kw), None) != 0 and 'workspace' in lib.n3d_last_error().decode()
        assert entry(None, None) != 0
    assert lib.n3d_attention(desc(Lq=0), None) == 0 and lib.n3d_attention(desc(B=0), None) == 0
    for kw, word in ((dict(Lq=0), 'queries'), (dict(lse=None), 'null'), (dict(dout=None), 'null'), (dict(dk=None), 'null'), (dict(dq=None, dk=None, dv=None), 'null'),
                     (dict(dout_strides=(128, 33, 16)), 'strides'), (dict(dout=4100), 'aligned'), (dict(dv=4100), 'aligned')):
        assert lib.n3d_attention_bwd(desc(workspace=4096, workspace_bytes=1 << 30, **kw), None) != 0 and word in lib.n3d_last_error().decode(), kw


def test_host_side_is_built_and_bound():
    """The C++ host side loads, is bound to the library's entry points, and reports the library's own refusals as RuntimeError (here: a launch that needs a
    device is refused by the library's argument checks before it gets that far)."""
    from next3d_amd import _lib
    ext = _lib.token_ext()
    assert ext is _lib.token_ext() and all(callable(getattr(ext, n)) for n in ('layer_norm', 'rotary', 'attention'))
    with pytest.raises(RuntimeError):
        ext.bind([0, 1])


def test_token_ops_refuse_sizes_and_lazy_values():
    from next3d_amd.torch_utils.ops.attention import attention
    from next3d_amd.torch_utils.ops.layer_norm import layer_norm
    from next3d_amd.torch_utils.ops.rotary import rotary
    one = torch.zeros(1)
    _raises('2\\^31', layer_norm, one.expand(1 << 31))
    _raises('2\\^31', rotary, one.expand(1 << 16, 1 << 15, 1, 2), one.int().expand(1 << 15, 1), (2,))
    half = one.half()
    for b, l in ((1 << 31, 1), (1, 1 << 31)):
        _raises('2\\^31', attention, half.expand(b, 1, 1, 8), half.expand(b, l, 1, 8), half.expand(b, l, 1, 8))
    x = torch._neg_view(torch.ones(2, 8))                              # a view whose memory holds the negated values
    _raises('dense', layer_norm, x)
    _raises('dense', layer_norm, torch.ones(2, 8), x[0])
    _raises('dense', rotary, x.view(1, 2, 1, 8), torch.zeros(2, 1), (8,))
    q = torch.zeros(1, 2, 1, 8).half()
    _raises('dense', attention, q, torch._neg_view(q), q)
    for kw in (dict(softcap=5000.0), dict(softcap=1e-40), dict(softcap=float('nan')), dict(scale=1e38), dict(scale=-1e38)):
        _raises('finite', attention, q, q, q, **kw)


def test_attention_c_entries_refuse_sizes():
    from next3d_amd import _lib
    lib = _lib.lib()
    base = dict(q=4096, k=4096, v=4096, out=4096, lse=4096, dout=4096, dq=4096, dk=4096, dv=4096, scale=1.0, B=1, Lq=4, Lk=300, heads_q=1, heads_k=1, D=16, dtype=1,
                workspace=4096, workspace_bytes=1 << 60)
    for kw, word in ((dict(Lk=(1 << 30) + 1), 'rows'), (dict(Lq=(1 << 30) + 1), 'rows'), (dict(softcap=4097.0), 'softcap'), (dict(softcap=1e-35), 'softcap'),
                     (dict(scale=1e35), 'scale')):
        for entry in (lib.n3d_attention, lib.n3d_attention_bwd):
            assert entry(_lib.AttentionDesc(**dict(base, **kw)), None) != 0 and word in lib.n3d_last_error().decode(), kw
    many = _lib.AttentionDesc(**dict(base, B=1 << 10, Lq=1 << 19, heads_q=4, heads_k=4))
    assert lib.n3d_attention_bwd(many, None) != 0 and '2^31' in lib.n3d_last_error().decode()
    assert lib.n3d_attention_workspace(_lib.AttentionDesc(**dict(base, B=1 << 10, Lk=1 << 15, heads_q=64, heads_k=8))) >= 0      # (a large cache, single tokens)


def _host_side_calls():
    """Each operator's call of the C++ host side (no device check in front of it) and its floating-point arguments."""
    from next3d_amd import _lib
    ext = _lib.token_ext()
    pos, q, q16 = torch.zeros(3, 1), torch.ones(1, 3, 2, 8), torch.ones(1, 3, 2, 8).half()
    return (('layer_norm', lambda x, w, b: ext.layer_norm(x, w, b, 1e-5), [torch.ones(3, 8), torch.ones(8), torch.ones(8)]),
            ('rotary', lambda q, k, p: ext.rotary(q, k, p, (8,), 1e4, True, False)[0], [q, q, pos]),
            ('attention', lambda q, k, v, s: ext.attention(q, k, v, 1.0, False, None, None, None, None, 0.0, s, False)[0], [q16, q16, q16, torch.ones(2)]))


@pytest.mark.parametrize('op', [0, 1, 2])
def test_forward_mode_derivatives_are_refused(op):
    """A tangent on any argument: refused, not dropped."""
    import torch.autograd.forward_ad as fwd
    name, call, args = _host_side_calls()[op]
    for which in range(len(args)):
        with fwd.dual_level():
            duals = [fwd.make_dual(t, torch.ones_like(t)) if i == which else t for i, t in enumerate(args)]
            _raises(f'{name}: no forward-mode', call, *duals)


@pytest.mark.parametrize('op', [0, 1, 2])
def test_tracing_is_refused(op):
    """A tracer sees an empty tensor and not what fills it: refused, not recorded."""
    from torch.fx.experimental.proxy_tensor import make_fx
    name, call, args = _host_side_calls()[op]
    _raises(f'{name}: cannot be traced', torch.jit.trace, call, tuple(args))
    _raises(f'{name}: cannot be traced', make_fx(call), *args)


@pytest.mark.parametrize('op', [0, 1, 2])
def test_tensors_without_memory_are_refused(op):
    """A wrapping tensor holds no memory itself: refused, not taken for an absent argument."""
    class Wrapper(torch.Tensor):
        @staticmethod
        def __new__(cls, t):
            return torch.Tensor._make_wrapper_subclass(cls, t.shape, dtype=t.dtype, device=t.device)

        @classmethod
        def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
            return func(*(torch.zeros(a.shape, dtype=a.dtype) if isinstance(a, cls) else a for a in args), **(kwargs or {}))

    name, call, args = _host_side_calls()[op]
    for which in range(len(args)):
        _raises(f'{name}: a tensor without memory', call, *(Wrapper(t) if i == which else t for i, t in enumerate(args)))


def test_attention_c_entries_refuse_launches_of_2_to_the_32_threads():
    """HIP refuses such a launch; the library refuses the call before it enqueues anything.  One sequence fewer passes the same check."""
    from next3d_amd import _lib
    lib = _lib.lib()
    base = dict(q=4096, k=4096, v=4096, out=4096, lse=4096, dout=4096, dq=4096, dk=4096, dv=4096, scale=1.0, Lq=100, Lk=100, D=8, dtype=1)
    for kw, entries in ((dict(B=1 << 20, heads_q=16, heads_k=16), 'fb'), (dict(B=1 << 24, Lq=1, Lk=1, heads_q=1, heads_k=1), 'fb'), (dict(B=1 << 22, Lq=1, heads_q=16, heads_k=4), 'f'),
                        (dict(B=1 << 19, Lq=1, Lk=1000, heads_q=4, heads_k=4, D=8), 'b'), (dict(B=1 << 19, Lk=200, heads_q=8, heads_k=8, D=128), 'b')):
        for which in entries:
            entry, size = (lib.n3d_attention, lib.n3d_attention_workspace) if which == 'f' else (lib.n3d_attention_bwd, lib.n3d_attention_bwd_workspace)
            d = _lib.AttentionDesc(**dict(base, workspace=4096, workspace_bytes=1 << 60, **kw))
            assert entry(d, None) != 0 and 'one launch' in lib.n3d_last_error().decode(), (kw, which, lib.n3d_last_error())
            assert size(d) == -1 and 'one launch' in lib.n3d_last_error().decode()
            d.B -= 8
            assert size(d) >= 0, (kw, which)
    docs = _lib.AttentionDesc(**dict(base, B=1 << 23, Lq=1, Lk=300, heads_q=1, heads_k=1, q_documents=4096, k_documents=4096))
    assert lib.n3d_attention_bwd_workspace(docs) == -1 and 'one launch' in lib.n3d_last_error().decode()


def test_rotary_refuses_launches_of_2_to_the_32_threads():
    """Eight tokens a workgroup of 256 where a token has 256 pairs: 2^27 tokens are 2^24 workgroups."""
    from next3d_amd import _lib
    lib = _lib.lib()
    d = _lib.RotaryDesc(q=4096, positions=4096, out_q=4096, pos_token_stride=1, base=1e4, B=1 << 12, L=1 << 15, heads_q=1, D=512, axes=1, dtype=0)
    d.sections[0] = 512
    assert lib.n3d_rotary(d, None) != 0 and 'one launch' in lib.n3d_last_error().decode()


def test_rotary_refuses_sections_that_are_no_whole_numbers():
    from next3d_amd.torch_utils.ops.rotary import rotary
    q, pos = torch.zeros(2, 5, 3, 16), torch.zeros(5, 2, dtype=torch.int32)
    for sections in ((8.0, 8.0), (8.9, 7.9), ('8', 8), 16):
        _raises('whole numbers', rotary, q, pos, sections)
    _raises('HIP device only', rotary, q, pos, torch.tensor([8, 8]))


def test_tile_pieces_wait_for_their_descriptor(tmp_path):
    """A memory instruction may read a scalar register five wait states after a vector instruction wrote it; inside asm nobody but the asm sees to that."""
    import re
    from next3d_amd import build
    src, out = tmp_path / 'piece.hip', tmp_path / 'piece.s'
    src.write_text('''#include "attention.h"
__global__ void piece(const int* p, float* out) {
    __shared__ __align__(1024) float tile[4096];
    const int x = p[threadIdx.x], y = p[threadIdx.x + 64];
    for (int i = 0; i < 4; ++i) {
        const i32x4 r = {attn_uniform(x + i), attn_uniform(y) & 0xffff, attn_uniform(x ^ y), 0x00020000};
        attn_piece(r, x, attn_uniform(attn_lds(tile) + i * 1024));
        attn_piece(r, y, attn_uniform(attn_lds(tile) + y));
    }
    attn_sync();
    out[threadIdx.x] = tile[threadIdx.x];
}
''')
    subprocess.run([build.HIPCC, *build.CFLAGS, '-w', '-I', build.CSRC, '--cuda-device-only', '-S', str(src), '-o', str(out)], check=True, capture_output=True)

    def scalars(text):
        m = re.fullmatch(r's\[(\d+):(\d+)\]|s(\d+)', text)
        return set() if not m else {int(m.group(3))} if m.group(3) else set(range(int(m.group(1)), int(m.group(2)) + 1))

    at, written, pieces, vector_writes = 0, {}, 0, 0
    for line in out.read_text().splitlines():
        m = re.match(r'\s+([a-z]\w+)\s*([^;]*)', line)
        if not m:
            continue
        op, args = m.group(1), [a.strip() for a in m.group(2).split(',')]
        at += 1 + (int(args[0]) if op == 's_nop' else 0)
        if op.startswith('v_') or op.startswith('s_'):
            for r in scalars(args[0]):
                written[r] = at if op.startswith('v_') else -1000
                vector_writes += op == 'v_readfirstlane_b32'
        if op == 'buffer_load_dwordx4' and 'lds' in line:
            pieces += 1
            assert all(at - written.get(r, -1000) - 1 >= 5 for r in scalars(args[1])), line
    assert pieces == 8 and vector_writes >= 2


def test_host_side_belongs_to_one_torch(monkeypatch):
    """Loaded under another torch than it was built against, it is refused; under that torch the build's command is another one."""
    from next3d_amd import _lib, build
    assert _lib.token_ext().torch_version == torch.__version__
    command = build._ext_commands()[2]
    monkeypatch.setattr(torch, '__version__', '1.0.0')
    assert build._ext_commands()[2] != command
    monkeypatch.setattr(_lib, '_token_ext', None)
    _raises('built against torch', _lib.token_ext)


def test_objects_are_made_again_by_another_command(tmp_path):
    from next3d_amd import build
    obj = str(tmp_path / 'x.o')
    assert build._other_command(obj, ['hipcc', '-O3'])
    build._note_command(obj, ['hipcc', '-O3'])
    assert not build._other_command(obj, ['hipcc', '-O3']) and build._other_command(obj, ['hipcc', '-O2'])


def test_the_build_entry_compiles_every_time(monkeypatch):
    import __graft_entry__ as entry
    from next3d_amd import build
    asked = []
    monkeypatch.setattr(build, 'build', lambda force=False, verbose=True: asked.append(force) or build.LIB)
    entry.build()
    assert asked == [True]
