"""CPU: what the 8-bit blocks' and the embedding's entry points refuse, before any launch."""
import ctypes

import pytest
import torch

import kerneldev_amd as kd
from kerneldev_amd import _lib

P, NULL = 1 << 12, ctypes.c_void_p(0)  # an aligned address that the host never reads
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def _blocks(rows, cols, scale_rows):
    return kd.BlockFp8(torch.zeros(rows, cols).to(E4M3), torch.ones(scale_rows, -(-cols // 128)).to(E8M0))


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(4, 64).bfloat16(), torch.zeros(16, 64).bfloat16()
    for call in (lambda: kd.quantize_rows(x), lambda: kd.quantize_weight(w), lambda: kd.add_rms_norm_fp8(x, x),
                 lambda: kd.fp8_projection(x, w), lambda: kd.norm_projection(x, None, w), lambda: kd.swiglu_projection(x, x, w),
                 lambda: kd.embedding(torch.zeros(3, dtype=torch.int64), w),
                 lambda: kd.fp8_matmul(_blocks(4, 64, 4), _blocks(16, 64, 1))):
        with pytest.raises(ValueError, match="GPU"):
            call()


@pytest.mark.parametrize("text,call", [
    ("multiple of 16", lambda x, w: kd.quantize_rows(x[:, :24])),
    ("multiple of 16", lambda x, w: kd.quantize_weight(w[:, :56])),
    ("must be \\[N, K\\]", lambda x, w: kd.quantize_weight(w[0])),
    ("multiple of 16", lambda x, w: kd.add_rms_norm_fp8(x[:, :24])),
    ("multiple of 8", lambda x, w: kd.norm_projection(x[:, :20], None, w[:, :20])),
    ("at most 8192", lambda x, w: kd.add_rms_norm_fp8(torch.zeros(1, 8208).bfloat16())),
    ("one shape, type", lambda x, w: kd.add_rms_norm_fp8(x, x[:2])),
    ("one shape, type", lambda x, w: kd.add_rms_norm_fp8(x, x.half())),
    ("bfloat16 or float16", lambda x, w: kd.add_rms_norm_fp8(x.float())),
    ("bfloat16 or float16", lambda x, w: kd.fp8_projection(x.float(), w.float())),
    ("1 to 4 weights", lambda x, w: kd.norm_projection(x, None)),
    ("1 to 4 weights", lambda x, w: kd.norm_projection(x, None, w, w, w, w, w)),
    ("a weight must be", lambda x, w: kd.fp8_projection(x, w[:, :56])),
    ("a weight must be", lambda x, w: kd.fp8_projection(x, w[:12])),
    ("type and device", lambda x, w: kd.fp8_projection(x, w.half())),
    ("one shape, type", lambda x, w: kd.swiglu_projection(x, x[:3], w)),
    ("at least one dimension", lambda x, w: kd.quantize_rows(x[0, 0])),
    ("float8_e4m3fn", lambda x, w: kd.fp8_matmul((x, x), (w, w))),
    ("multiple of 16", lambda x, w: kd.fp8_matmul(_blocks(4, 24, 4), _blocks(16, 24, 1))),
    ("expected", lambda x, w: kd.fp8_matmul(_blocks(4, 64, 4), _blocks(16, 48, 1))),
    ("do not belong", lambda x, w: kd.fp8_matmul(_blocks(4, 64, 3), _blocks(16, 64, 1))),
    ("do not belong", lambda x, w: kd.fp8_matmul(_blocks(4, 64, 4), _blocks(16, 64, 16))),
    ("out_dtype", lambda x, w: kd.fp8_matmul(_blocks(4, 64, 4), _blocks(16, 64, 1), torch.float64)),
    ("do not belong", lambda x, w: kd.dequantize((torch.zeros(4, 64).to(E4M3), torch.ones(4, 2).to(E8M0)))),
    ("int64 or int32", lambda x, w: kd.embedding(torch.zeros(3), w)),
    ("\\[V, D\\]", lambda x, w: kd.embedding(torch.zeros(3, dtype=torch.int64), w[0])),
    ("bf16, fp16 or fp32", lambda x, w: kd.embedding(torch.zeros(3, dtype=torch.int64), w.double())),
    ("padding_idx", lambda x, w: kd.embedding(torch.zeros(3, dtype=torch.int64), w, padding_idx=16)),
])
def test_bad_arguments_raise(text, call):
    with pytest.raises(ValueError, match=text):
        call(torch.zeros(4, 64).bfloat16(), torch.zeros(16, 64).bfloat16())


def test_dequantize_runs_anywhere():
    w = kd.BlockFp8(torch.full((130, 144), 3.0).to(E4M3), torch.tensor([[2.0, 4.0], [8.0, 0.5]]).to(E8M0))
    v = kd.dequantize(w)
    assert v[0, 0] == 6 and v[0, 143] == 12 and v[129, 127] == 24 and v[128, 128] == 1.5


def _set(args, **values):
    for k, v in values.items():
        if isinstance(v, (list, tuple)):
            field = getattr(args, k)
            for i, x in enumerate(v):
                field[i] = x
        else:
            setattr(args, k, v)
    return args


GOOD = {
    "kd_quant_rows8": (_lib.Rows8Args, dict(x=[P], x_stride=[64], cols=[64], n=1, dtype=0, rows=4, y=P, y_stride=64, scale=P,
                                            total=64)),
    "kd_quant_weight8": (_lib.Weight8Args, dict(w=[P], w_stride=[64], rows=[16], n=1, dtype=0, K=64, total=16, y=P, y_stride=64,
                                                scale=P, yt=P, yt_stride=16, scale_t=P)),
    "kd_matmul8": (_lib.Matmul8Args, dict(a=P, b=P, lda=64, ldb=64, a_scale=P, b_scale=P, out=P, ldo=16, M=4, N=16, K=64, dtype=0)),
    "kd_norm8": (_lib.Norm8Args, dict(x=P, delta=P, sum=P, y=P, y_stride=64, scale=P, rstd=P, rows=4, D=64, dtype=0, eps=1e-6)),
    "kd_norm8_bwd": (_lib.Norm8BwdArgs, dict(g=P, ds=P, y=P, y_stride=64, scale=P, rstd=P, dx=P, rows=4, D=64, dtype=0)),
    "kd_gate8": (_lib.Gate8Args, dict(a=P, b=P, a_stride=64, b_stride=64, y8=P, y_scale=P, a8=P, a_scale=P, b8=P, b_scale=P,
                                      stride=64, rows=4, H=64, dtype=0)),
    "kd_gate8_bwd": (_lib.Gate8Args, dict(dy=P, da=P, db=P, a8=P, a_scale=P, b8=P, b_scale=P, stride=64, rows=4, H=64, dtype=0)),
    "kd_weight_grad8": (_lib.Wgrad8Args, dict(dy=[P], ldy=[16], cols=[16], n=1, x=P, ldx=64, x_scale=P, dw=P, ws=P, ws_bytes=1 << 40, M=4, N=16,
                                              K=64, dtype=0)),
    "kd_embed": (_lib.EmbedArgs, dict(tokens=P, n=5, weight=P, out=P, vocab=7, dim=16, padding_idx=-1, tokens_dtype=0, dtype=0)),
    "kd_embed_grad": (_lib.EmbedArgs, dict(tokens=P, n=5, dy=P, dw=P, vocab=7, dim=16, padding_idx=-1, tokens_dtype=0, dtype=0)),
}
INVALID, UNSUPPORTED = _lib.KD_ERR_INVALID, _lib.KD_ERR_UNSUPPORTED


@pytest.mark.parametrize("name,change,code", [
    ("kd_quant_rows8", dict(n=0), INVALID), ("kd_quant_rows8", dict(n=5), INVALID), ("kd_quant_rows8", dict(dtype=3), UNSUPPORTED),
    ("kd_quant_rows8", dict(cols=[60], total=60), UNSUPPORTED), ("kd_quant_rows8", dict(total=72), INVALID),
    ("kd_quant_rows8", dict(x=[P + 8]), INVALID), ("kd_quant_rows8", dict(x_stride=[56]), INVALID),
    ("kd_quant_rows8", dict(x_stride=[68]), INVALID), ("kd_quant_rows8", dict(y_stride=48), INVALID),
    ("kd_quant_rows8", dict(y_stride=72), INVALID), ("kd_quant_rows8", dict(y=None), INVALID),
    ("kd_quant_rows8", dict(scale=None), INVALID), ("kd_quant_rows8", dict(rows=0), INVALID),
    ("kd_quant_rows8", dict(n=2, x=[P, P], x_stride=[64, 64], cols=[64, 64], total=128), INVALID),
    ("kd_quant_weight8", dict(rows=[12], total=12), UNSUPPORTED), ("kd_quant_weight8", dict(K=60), UNSUPPORTED),
    ("kd_quant_weight8", dict(scale_t=None), INVALID), ("kd_quant_weight8", dict(yt_stride=8), INVALID),
    ("kd_quant_weight8", dict(n=2, w=[P, P], w_stride=[64, 64], rows=[16, 16], total=32), INVALID),
    ("kd_matmul8", dict(K=24), UNSUPPORTED), ("kd_matmul8", dict(K=0), UNSUPPORTED), ("kd_matmul8", dict(M=0), INVALID),
    ("kd_matmul8", dict(lda=48), INVALID), ("kd_matmul8", dict(lda=72), INVALID), ("kd_matmul8", dict(a=P + 8), INVALID),
    ("kd_matmul8", dict(a_scale=None), INVALID), ("kd_matmul8", dict(ldo=15), INVALID), ("kd_matmul8", dict(dtype=4), UNSUPPORTED),
    ("kd_matmul8", dict(M=1 << 30), UNSUPPORTED), ("kd_quant_weight8", dict(rows=[1 << 22], total=1 << 22, K=1 << 22, w_stride=[1 << 22], y_stride=1 << 22), UNSUPPORTED),
    ("kd_matmul8", dict(lda=1 << 24, ldb=1 << 24), INVALID), ("kd_matmul8", dict(M=(1 << 31) - 1, N=(1 << 31) - 1, ldo=1 << 31), UNSUPPORTED),
    ("kd_norm8", dict(D=60), UNSUPPORTED), ("kd_norm8", dict(D=8200), UNSUPPORTED), ("kd_norm8", dict(dtype=2), UNSUPPORTED),
    ("kd_norm8", dict(sum=None), INVALID), ("kd_norm8", dict(x=P + 2), INVALID), ("kd_norm8", dict(y_stride=48), INVALID),
    ("kd_norm8", dict(rows=(1 << 32) + 1), INVALID),
    ("kd_norm8_bwd", dict(rstd=None), INVALID), ("kd_norm8_bwd", dict(dx=None), INVALID), ("kd_norm8_bwd", dict(ds=P + 4), INVALID),
    ("kd_gate8", dict(H=60), UNSUPPORTED), ("kd_gate8", dict(a_stride=56), INVALID), ("kd_gate8", dict(b8=None), INVALID),
    ("kd_gate8", dict(y_scale=None), INVALID), ("kd_gate8_bwd", dict(a8=None), INVALID), ("kd_gate8_bwd", dict(da=P + 2), INVALID),
    ("kd_weight_grad8", dict(N=12), UNSUPPORTED), ("kd_weight_grad8", dict(N=24), INVALID), ("kd_weight_grad8", dict(n=0), INVALID),
    ("kd_weight_grad8", dict(n=2, dy=[P, P], ldy=[16, 16], cols=[16, 16], N=32), INVALID), ("kd_weight_grad8", dict(M=0), INVALID), ("kd_weight_grad8", dict(M=(1 << 31) - 1), UNSUPPORTED),
    ("kd_weight_grad8", dict(ws_bytes=16), INVALID),
    ("kd_weight_grad8", dict(ldy=[12]), INVALID), ("kd_weight_grad8", dict(dy=[P + 8]), INVALID), ("kd_weight_grad8", dict(dtype=2), UNSUPPORTED), ("kd_weight_grad8", dict(x_scale=None), INVALID),
    ("kd_embed", dict(n=0), UNSUPPORTED), ("kd_embed", dict(vocab=0), UNSUPPORTED), ("kd_embed", dict(dim=0), UNSUPPORTED),
    ("kd_embed", dict(tokens=None), INVALID), ("kd_embed", dict(tokens_dtype=2), INVALID), ("kd_embed", dict(dtype=3), UNSUPPORTED),
    ("kd_embed", dict(weight=None), INVALID), ("kd_embed_grad", dict(dy=None), INVALID), ("kd_embed_grad", dict(dw=P + 2), INVALID),
    ("kd_embed_grad", dict(n=1 << 31), UNSUPPORTED), ("kd_embed_grad", dict(vocab=1 << 31), UNSUPPORTED),
    ("kd_embed_grad", dict(n=(1 << 31) - 1, dim=1 << 20), UNSUPPORTED),
])
def test_c_abi_refusals(name, change, code):
    struct, good = GOOD[name]
    args = _set(_set(struct(), **good), **change)
    fn = getattr(_lib.load(), name)
    more = (ctypes.c_void_p(P), 1 << 40) if name == "kd_embed_grad" else ()
    assert fn(ctypes.byref(args), *more, NULL) == code, _lib.load().kd_last_error_string()


def test_c_abi_null_and_workspaces():
    lib = _lib.load()
    for name in GOOD:
        more = (NULL, 0) if name == "kd_embed_grad" else ()
        assert getattr(lib, name)(None, *more, NULL) == INVALID
    args = _set(_lib.EmbedArgs(), **GOOD["kd_embed_grad"][1])
    need = lib.kd_embed_grad_ws_bytes(5, 7, 16)
    assert need > 0 and lib.kd_embed_grad(ctypes.byref(args), ctypes.c_void_p(P), need - 1, NULL) == INVALID
    assert lib.kd_embed_grad(ctypes.byref(args), ctypes.c_void_p(P + 8), need, NULL) == INVALID
    for bad in ((0, 7, 16), (5, 0, 16), (5, 7, 0), (1 << 31, 7, 16)):
        assert lib.kd_embed_grad_ws_bytes(*bad) == -1
    assert lib.kd_weight_grad8_ws_bytes(4, 12, 64, 0) == -1 and lib.kd_weight_grad8_ws_bytes(4, 16, 64, 0) >= 4 * 16 * 64
