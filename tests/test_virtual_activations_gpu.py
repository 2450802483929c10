"""KrnEngine.activations() returns the forward state that the pass itself uses: the virtual tensors (blocks 2-4, recomputed in float32 by every kernel that
reads them) unrounded, everything else as it is stored."""
import ctypes as C

import pytest
import torch

pytestmark = pytest.mark.gpu

from oracle import krn_oracle as O  # noqa: E402
from speedplusbaseline_amd import _lib as L  # noqa: E402
from speedplusbaseline_amd.engine import KrnEngine  # noqa: E402

B = 48


@pytest.mark.parametrize("precision", ["bf16", "fp16", "fp32"])
def test_virtual_tensors_are_not_rounded(device, precision):
    x, y = O.synth_batch(B)
    eng = KrnEngine(11).attach(device, precision)
    sd = O.init_state(11)
    for info in eng.param_infos:
        eng.param_view(info).copy_(sd[info[0]].to(device))
    for name, shape, off, numel in eng.buffer_infos:
        eng.buffers[off: off + numel].view(shape).copy_(sd[name].to(device))
    eng.forward(x.to(device), y.to(device), training=True)
    acts = eng.activations(B)
    virtual = eng.virtual_activations(B)
    if precision == "fp32":
        assert virtual == [] and all(v.dtype == torch.float32 for v in acts.values())
        return
    t = torch.bfloat16 if precision == "bf16" else torch.float16
    assert virtual == ["base.2.conv.0.1", "base.3.conv.0.1", "base.4.conv.0.1"]
    # the same tensors rounded to the storage type, in their workspace slots
    h, ws = eng._ctx[(B, 0)]
    L.check(eng.lib.spb_krn_ctx_materialize(h, None), "spb_krn_ctx_materialize")
    torch.cuda.synchronize()
    ai, seen = L.ActInfo(), 0
    for a in range(eng.lib.spb_krn_num_acts(eng.h)):
        L.check(eng.lib.spb_krn_ctx_act_info(h, a, C.byref(ai)), "spb_krn_ctx_act_info")
        name = eng.bn_names[ai.bn_index][: -len(".num_batches_tracked")]
        z = acts[name]
        if name not in virtual:
            assert z.dtype == t, name
            continue
        seen += 1
        n = B * ai.H * ai.W * ai.C
        stored = ws[ai.z_off: ai.z_off + 2 * n].view(t).view(B, ai.H, ai.W, ai.C).permute(0, 3, 1, 2)
        assert z.dtype == torch.float32 and z.shape == stored.shape
        # a product of 16 or 24 terms in float32 and its rounding: half a step of the type (float16's subnormal step 2^-24 below 2^-14), and the sums'
        # own roundings, 24 * 2^-24 of their terms, which are below 2^5 here
        zd, sd_ = z.double(), stored.double()
        lim = torch.finfo(t).eps / 2 * zd.abs() * (1 + 2.0 ** -8) + (2.0 ** -25 if t == torch.float16 else 0) + 24 * 2.0 ** -24 * 32
        assert ((zd - sd_).abs() <= lim).all()
        assert (z != z.to(t).float()).double().mean() > 0.9
    assert seen == 3
    # refusals: not a virtual tensor, too little room, no output
    out = torch.empty(8, device=device)
    first = [a for a in range(eng.lib.spb_krn_num_acts(eng.h)) if eng.lib.spb_krn_ctx_virtual(h, a) == 1][0]
    for args in ((0, C.c_void_p(out.data_ptr()), 1 << 40), (first, C.c_void_p(out.data_ptr()), 8), (first, None, 1 << 40), (-1, C.c_void_p(out.data_ptr()), 1 << 40)):
        assert eng.lib.spb_krn_ctx_virtual_z(h, *args, None) == -1
