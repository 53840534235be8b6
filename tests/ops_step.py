"""The single-token form of span attention through the C ABI."""
import ctypes as C

import torch


def step_with_lse(q, k, v, lo, hi, heads, kv_heads, scale, cap=0.0, slopes=None, max_keys=1):
    """nmtgan_attn_span_step with its lse, which the function of tensors does not hand out."""
    from nmt_gan_amd import _lib as L
    m, dh = q.shape[0], q.shape[1] // heads
    out = torch.full_like(q, 7.0)
    lse = torch.full((m, heads), 7.0, device=q.device)
    a = L.SpanArgs(dtype={torch.bfloat16: L.NMTGAN_BF16, torch.float16: L.NMTGAN_F16, torch.float32: L.NMTGAN_F32}[q.dtype], M=m,
                   N=k.shape[0], heads=heads, kv_heads=kv_heads, dh=dh, q=q.data_ptr(), ldq=q.stride(0), k=k.data_ptr(), ldk=k.stride(0),
                   v=v.data_ptr(), ldv=v.stride(0), lo=lo.data_ptr(), hi=hi.data_ptr(), slopes=None if slopes is None else slopes.data_ptr(),
                   scale=scale, cap=cap, out=out.data_ptr(), ldo=out.stride(0), lse=lse.data_ptr())
    need = L.lib.nmtgan_attn_span_step_workspace_bytes(m, heads, kv_heads, dh, max_keys)
    ws = torch.empty(max(need, 1), dtype=torch.uint8, device=q.device)
    L.check(L.lib.nmtgan_attn_span_step(C.byref(a), max_keys, ws.data_ptr() if need else None, need, L.stream_ptr()), "step")
    torch.cuda.synchronize()
    return out, lse
