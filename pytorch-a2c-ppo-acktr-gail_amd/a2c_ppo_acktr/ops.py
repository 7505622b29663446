"""Tensor-level wrappers over the C-ABI operators (include/acktr_hip.h).

Thin plumbing only: shape checks on the host (a wrong shape must never reach a
kernel), device pointers + the current stream handed to the library.  Every
function requires fp32 contiguous GPU tensors and raises otherwise; the gated
core's operators at the end take bf16, fp16 or fp32 and rows of wider tensors.
"""
import contextlib
import ctypes
import gc
import torch

from . import _hip

f32 = torch.float32
_ws_cache = {}
WS_MIN_BYTES = 1 << 20
_ws_retired = []          # outgrown buffers, kept alive for captured graphs that still point into them

# Optional per-launch timing with HIP events on the launch stream (used by bench.py for the roofline
# figures).  `profiler` is None (off) or a dict name -> list of (start_event, end_event, work) tuples.
profiler = None


class _Timed(object):
    __slots__ = ('name', 'work', 'ev')

    def __init__(self, name, work):
        self.name, self.work = name, work

    def __enter__(self):
        if profiler is not None:
            s = torch.cuda.Event(enable_timing=True)
            s.record()
            self.ev = s
        return self

    def __exit__(self, *a):
        if profiler is not None:
            e = torch.cuda.Event(enable_timing=True)
            e.record()
            profiler.setdefault(self.name, []).append((self.ev, e, self.work))
        return False


def profile_summary():
    """name -> dict(calls, avg_ms, total_ms, flops_per_call) after a device sync."""
    out = {}
    if profiler is None:
        return out
    torch.cuda.synchronize()
    for name, recs in profiler.items():
        ms = [s.elapsed_time(e) for s, e, _ in recs]
        # an event bracket also counts GPU idle time when the host is late with the launch inside it (one 35 ms host
        # stall once turned a 78 us kernel into a 2.2 ms "average"): brackets above 3x the median are left out
        med = sorted(ms)[len(ms) // 2]
        kept = [m for m in ms if m <= 3.0 * med] or ms
        out[name] = dict(calls=len(ms), avg_ms=sum(kept) / len(kept), total_ms=sum(kept) / len(kept) * len(ms),
                         flops_per_call=sum(w for _, _, w in recs) / len(recs), outliers_dropped=len(ms) - len(kept))
    return out


def workspace(device, nbytes, tag='ws'):
    """Per-(device, tag) scratch buffer, grown on demand and reused across calls.

    A buffer that is outgrown is RETIRED, never freed: hipGraphs captured earlier (PPO / A2C / ACKTR / GAIL steps)
    hold raw pointers into it and keep replaying while another agent with larger shapes makes this cache grow.
    Growth is at least 2x, so the retired buffers of a tag add up to less than its live one."""
    key = (str(device), tag)
    buf = _ws_cache.get(key)
    if buf is None or buf.numel() < nbytes:
        if buf is not None:
            _ws_retired.append(buf)
        want = max(int(nbytes), WS_MIN_BYTES, 2 * buf.numel() if buf is not None else 0)
        buf = torch.empty(want, dtype=torch.uint8, device=device)
        _ws_cache[key] = buf
    # exactly the bytes asked for: several entry points cut their reduction into as many split-K slabs as the workspace
    # they are GIVEN holds, so handing over the whole (grown) buffer made results depend on what had run before in the
    # process -- by one rounding, which a ReLU gate at zero can turn into another trajectory (tests/test_u8_gpu.py)
    return buf[:nbytes] if nbytes < buf.numel() else buf


@contextlib.contextmanager
def graph_capture(g, **kw):
    """`with torch.cuda.graph(g)` with Python's cyclic garbage collector OFF for the duration.  torch collects once on
    entry, but a collection that the allocation counters trigger DURING the capture can still finalise an unreachable
    torch.cuda.CUDAGraph (a dropped agent's, kept alive until then by a reference cycle): its destructor calls into HIP,
    which answers "operation not permitted when stream is capturing", and torch aborts the process from the destructor
    (seen once in the GPU suite, inside the GAIL step's capture)."""
    was_enabled = gc.isenabled()
    gc.disable()                # (torch.cuda.graph collects explicitly on entry; a second full collection here cost the
                                #  bench's ACKTR loop, whose capture falls into its timed updates, 110 ms)
    try:
        with torch.cuda.graph(g, **kw):
            yield g
    finally:
        if was_enabled:
            gc.enable()


def _p(t, name, dtype=f32):
    return _hip.dev_ptr(t, dtype, name)


def _conv_out(H, K, S):
    return (H - K) // S + 1


def _pack_layout(layers, B):
    """[(key, byte offset, bytes, job tuple)] of the weight-image workspaces inside ONE buffer (256-byte aligned slots),
    and the buffer size.  Layers the stationary kernels do not cover are left out."""
    L = _hip.lib()
    out, off = [], 0
    for key, w, stride, hw, dgrad in layers:
        OC, C, KH, KW = w.shape
        if dgrad:
            nb = L.acktr_conv2d_dgrad_workspace_bytes(B, C, hw, hw, OC, KH, KW, stride)
        else:
            nb = L.acktr_conv2d_fwd_workspace_bytes(C, hw, hw, OC, KH, KW, stride)
        if not nb or (w.data_ptr() & 15):
            continue
        out.append((key, off, int(nb), (C, hw, OC, KH, KW, stride, 1 if dgrad else 0)))
        off += (int(nb) + 255) // 256 * 256
    return out, off


def _pack_jobs(layout, weights, buf):
    jobs = [_hip.ConvPackJob(weights[key].data_ptr(), buf.data_ptr() + off, nb, C, hw, hw, OC, KH, KW, stride, dg)
            for key, off, nb, (C, hw, OC, KH, KW, stride, dg) in layout]
    return (_hip.ConvPackJob * len(jobs))(*jobs)


def _run_pack(layout, weights, buf, stream_dev):
    arr = _pack_jobs(layout, weights, buf)
    return _hip.lib().acktr_conv2d_pack_weights_f32(arr, len(arr), _hip.cur_stream(stream_dev))


def pack_conv_weights(layers, B, cache, trust=False):
    """Re-ordered weights of several conv layers in ONE launch.  layers: list of (key, w, stride, in_hw, dgrad); the
    result maps key -> workspace tensor to hand to conv2d_fwd / conv2d_dgrad as `packed`.  Layers the stationary
    kernels do not cover are left out (those entry points then prepare their weights themselves).  `cache` (a dict
    owned by the policy) keeps the workspaces: they must survive from a forward to its backward, so they cannot be
    the process-wide scratch buffers.  All workspaces are slots of ONE buffer, so that an optimiser can keep the images
    in step with the parameters through one offset table (conv_image_map).
    trust=True: the images are known to be current (the caller re-packed at the start of its update and its optimiser
    steps write the images themselves): no launch."""
    if not layers:
        return {}
    dev = layers[0][1].device
    wptr = layers[0][1].data_ptr()
    if cache.get('_jobs') is not None and cache.get('_B', 0) >= B and cache.get('_wptr') == wptr and cache['_buf'].device == dev:
        # the common case, without the host work of laying the buffer out again (it showed as GPU idle time in front of
        # every update's first graph launch): same parameters, a batch the buffer already covers
        if not trust:
            if _hip.lib().acktr_conv2d_pack_weights_f32(cache['_jobs'], len(cache['_jobs']), _hip.cur_stream(dev)) != 0:
                return {}
        return cache['_views']
    # sized for the largest batch seen so far: a smaller batch (Policy.act between two updates) uses the front of the same
    # slots, so captured graphs that hold pointers into the buffer stay valid; an outgrown buffer is retired, not freed
    B = max(int(B), cache.get('_B', 0) if cache.get('_buf') is not None and cache['_buf'].device == dev else 0)
    layout, total = _pack_layout(layers, B)
    if not layout:
        return {}
    sig = tuple((k, o, n) for k, o, n, _ in layout)
    buf = cache.get('_buf')
    fresh = buf is None or buf.device != dev or cache.get('_sig') != sig
    if fresh:
        if buf is not None:
            _ws_retired.append(buf)
        cache['_B'] = B
        # zeroed: behind the weight image a dgrad workspace holds the zero-padded dY planes, whose borders nobody
        # writes when the producer of dY fills the interiors itself (padded_dy_view / conv2d_dgrad(dy_prepadded))
        buf = torch.zeros(total, dtype=torch.uint8, device=dev)
        cache['_buf'], cache['_sig'], cache['_map'] = buf, sig, None
        cache['_views'] = {k: buf[o:o + n] for k, o, n, _ in layout}
    weights = {key: w for key, w, _, _, _ in layers}
    if fresh or not trust:
        if _run_pack(layout, weights, buf, dev) != 0:      # a layer outside the stationary kernels' shapes
            return {}
    cache['_jobs'] = _pack_jobs(layout, weights, buf)
    cache['_wptr'] = wptr
    return cache['_views']


def conv_image_map(layers, B, cache, offset_of):
    """_hip.PackMap for an optimiser that stores conv weights to their weight-image slots as it updates them
    (acktr_clip_adam_dev_pack_f32), or None.  offset_of(w) -> float offset of parameter w in the flat buffer.  The
    tables come from the pack kernel itself: it is run once on weights that hold their own element number, and every
    image slot then says which parameter element it wants."""
    if cache.get('_map') is not None and cache.get('_jobs') is not None and cache.get('_B', 0) >= B:
        return cache['_map'][0]
    if not pack_conv_weights(layers, B, cache, trust=True):
        return None
    if cache.get('_map') is not None:
        return cache['_map'][0]
    dev = cache['_buf'].device
    layout, total = _pack_layout(layers, cache['_B'])
    by_key = {key: w for key, w, _, _, _ in layers}
    lo = min(offset_of(w) for w in by_key.values())
    hi = max(offset_of(w) + w.numel() for w in by_key.values())
    idx_w = {key: (torch.arange(1, w.numel() + 1, dtype=torch.float32, device=dev).view(w.shape).contiguous())
             for key, w in by_key.items()}
    if max(w.numel() for w in by_key.values()) >= (1 << 24):
        return None
    tmp = torch.zeros(total, dtype=torch.uint8, device=dev)
    if _run_pack(layout, idx_w, tmp, dev) != 0:
        return None
    img = tmp.view(torch.float32)
    t = [torch.full((hi - lo,), -1, dtype=torch.int32, device=dev) for _ in range(2)]
    for key, off, nb, job in layout:
        region = img[off // 4:(off + nb) // 4]
        slots = region.nonzero().view(-1)
        elems = region[slots].long() - 1 + (offset_of(by_key[key]) - lo)
        which = t[1] if job[-1] else t[0]
        if bool((which[elems] >= 0).any()):
            return None                        # two images of one kind want the same parameter: not a layout this map covers
        which[elems] = (slots + off // 4).to(torch.int32)
    pm = _hip.PackMap(lo, hi, t[0].data_ptr(), t[1].data_ptr(), cache['_buf'].data_ptr())
    cache['_map'] = (pm, t)                    # (the tables stay alive with the cache)
    return pm


def gate_mask_like(B, OC, OH, OW, device):
    """Buffer for the ReLU gate of a [B,OC,OH,OW] conv output as bits (acktr_conv2d_gate_mask_bytes)."""
    nb = _hip.lib().acktr_conv2d_gate_mask_bytes(B, OC, OH, OW)
    return torch.empty(nb // 4, dtype=torch.int32, device=device)


def conv2d_fwd(x, w, bias, stride, in_scale=1.0, relu=True, gather_idx=None, out=None, packed=None, gate_mask=None):
    """y = relu?(in_scale*conv2d(x[gather_idx], w) + bias); x [Bsrc,C,H,W], w [OC,C,KH,KW].
    gate_mask (int32 words, gate_mask_like): also receives (y > 0) as bits for conv2d_dgrad(gate_bits=) of the next
    layer -- the 8x8 stride-4 layer on its stationary path only."""
    OC, C, KH, KW = w.shape
    H, W = x.shape[-2], x.shape[-1]
    assert x.shape[-3] == C, 'channel mismatch'
    B = x.shape[0] if gather_idx is None else gather_idx.numel()
    OH, OW = _conv_out(H, KH, stride), _conv_out(W, KW, stride)
    if out is None:
        out = torch.empty(B, OC, OH, OW, dtype=f32, device=x.device)
    assert out.shape == (B, OC, OH, OW)
    L = _hip.lib()
    nb = L.acktr_conv2d_fwd_workspace_bytes(C, H, W, OC, KH, KW, stride)
    ws = packed if packed is not None else (workspace(x.device, nb, tag='convfwd') if nb else None)
    if x.dtype == torch.uint8:             # frames kept as bytes (RolloutStorage(obs_dtype=torch.uint8)): conv1 only
        if (C, H, W, OC, KH, KW, stride) != (4, 84, 84, 32, 8, 8, 4) or ws is None:
            raise RuntimeError('uint8 inputs are supported for the first NatureCNN layer only (4x84x84, 32 filters 8x8 s4)')
        with _Timed('conv%ds%d_fwd' % (KH, stride), 2.0 * B * OH * OW * OC * C * KH * KW):
            args = (_p(x, 'x', torch.uint8), _p(gather_idx, 'gather_idx', torch.int64), _p(w, 'w'),
                    _p(bias, 'bias'), _p(out, 'y'), B, float(in_scale), 1 if relu else 0,
                    _p(ws, 'workspace', torch.uint8), ws.numel(), 1 if packed is not None else 0)
            if gate_mask is not None:
                assert gate_mask.numel() * 4 >= L.acktr_conv2d_gate_mask_bytes(B, OC, OH, OW)
                rc = L.acktr_conv1_fwd_u8_gate(*args, _p(gate_mask, 'gate_mask', torch.int32), _hip.cur_stream(x.device))
            else:
                rc = L.acktr_conv1_fwd_u8(*args, _hip.cur_stream(x.device))
        _hip.check(rc, 'acktr_conv1_fwd_u8')
        return out
    with _Timed('conv%ds%d_fwd' % (KH, stride), 2.0 * B * OH * OW * OC * C * KH * KW):
        args = (_p(x, 'x'), _p(gather_idx, 'gather_idx', torch.int64), _p(w, 'w'), _p(bias, 'bias'), _p(out, 'y'),
                B, C, H, W, OC, KH, KW, stride, float(in_scale), 1 if relu else 0,
                _p(ws, 'workspace', torch.uint8), ws.numel() if ws is not None else 0, 1 if packed is not None else 0)
        if gate_mask is not None:
            assert gate_mask.numel() * 4 >= L.acktr_conv2d_gate_mask_bytes(B, OC, OH, OW)
            rc = L.acktr_conv2d_fwd_gate_f32(*args, _p(gate_mask, 'gate_mask', torch.int32), _hip.cur_stream(x.device))
        else:
            rc = L.acktr_conv2d_fwd_f32(*args, _hip.cur_stream(x.device))
    _hip.check(rc, 'acktr_conv2d_fwd_f32')
    return out


def conv2d_wgrad(x, dy, w_shape, stride, dw, db=None, in_scale=1.0, gather_idx=None, pending=None):
    """pending (a _hip.SlabFin): the final slab sum may be left to the optimiser's norm launch
    (acktr_conv2d_wgrad_deferred_f32); pending.dst is None afterwards when the call completed on its own.  The slabs
    live in the shared workspace: nothing else may use it before that optimiser call."""
    OC, C, KH, KW = w_shape
    H, W = x.shape[-2], x.shape[-1]
    B = dy.shape[0]
    assert dy.shape == (B, OC, _conv_out(H, KH, stride), _conv_out(W, KW, stride))
    assert dw.numel() == OC * C * KH * KW and (db is None or db.numel() == OC)
    if gather_idx is None:
        assert x.shape[0] == B
    else:
        assert gather_idx.numel() == B
    L = _hip.lib()
    if x.dtype == torch.uint8:
        if (C, H, W, OC, KH, KW, stride) != (4, 84, 84, 32, 8, 8, 4):
            raise RuntimeError('uint8 inputs are supported for the first NatureCNN layer only (4x84x84, 32 filters 8x8 s4)')
        ws = workspace(x.device, L.acktr_conv1_wgrad_u8_workspace_bytes(B))
        with _Timed('conv%ds%d_wgrad' % (KH, stride), 2.0 * dy[0].numel() * B * C * KH * KW):
            rc = L.acktr_conv1_wgrad_u8(_p(x, 'x', torch.uint8), _p(gather_idx, 'gather_idx', torch.int64), _p(dy, 'dy'),
                                        _p(dw, 'dw'), _p(db, 'db'), B, float(in_scale), _p(ws, 'workspace', torch.uint8),
                                        ws.numel(), ctypes.byref(pending) if pending is not None else None,
                                        _hip.cur_stream(x.device))
        _hip.check(rc, 'acktr_conv1_wgrad_u8')
        return
    nbytes = L.acktr_conv2d_wgrad_workspace_bytes(B, C, H, W, OC, KH, KW, stride)
    ws = workspace(x.device, nbytes)
    with _Timed('conv%ds%d_wgrad' % (KH, stride), 2.0 * dy[0].numel() * B * C * KH * KW):
        if pending is not None:
            rc = L.acktr_conv2d_wgrad_deferred_f32(
                _p(x, 'x'), _p(gather_idx, 'gather_idx', torch.int64), _p(dy, 'dy'), _p(dw, 'dw'), _p(db, 'db'),
                B, C, H, W, OC, KH, KW, stride, float(in_scale), _p(ws, 'workspace', torch.uint8), ws.numel(),
                ctypes.byref(pending), _hip.cur_stream(x.device))
        else:
            rc = L.acktr_conv2d_wgrad_f32(
                _p(x, 'x'), _p(gather_idx, 'gather_idx', torch.int64), _p(dy, 'dy'), _p(dw, 'dw'), _p(db, 'db'),
                B, C, H, W, OC, KH, KW, stride, float(in_scale), _p(ws, 'workspace', torch.uint8), ws.numel(),
                _hip.cur_stream(x.device))
    _hip.check(rc, 'acktr_conv2d_wgrad_f32')


def padded_dy_view(packed, B, w, stride, in_hw):
    """The zero-padded dY region ([B, OC, 11, 11] fp32) inside a stationary-dgrad workspace from pack_conv_weights, or
    None.  A producer of that layer's dY (linear_dgrad / conv2d_dgrad with padded_out=) writes the interiors there and
    conv2d_dgrad(..., dy_prepadded=True) then skips its padding pass; the borders stay zero from the allocation."""
    if packed is None:
        return None
    OC, C, KH, KW = w.shape
    off = _hip.lib().acktr_conv2d_dgrad_padded_dy_offset_bytes(C, in_hw, in_hw, OC, KH, KW, stride)
    n = B * OC * 121
    if off < 0 or off % 4 or packed.numel() < off + 4 * n:
        return None
    return packed[off:off + 4 * n].view(f32).view(B, OC, 11, 11)


def conv2d_dgrad(dy, w, x_act, stride, out=None, packed=None, dy_prepadded=False, padded_out=None, carry=None,
                 gate_bits=None):
    """dx = conv_transpose(dy, w) * (x_act > 0); x_act [B,C,H,W] is the (post-ReLU) input of the layer.
    dy_prepadded: `packed` already holds this dY zero-padded (see padded_dy_view); padded_out [B,C,H+2p,W+2p]: dx is
    also written there, interior only.  carry (a _hip.SlabFin left pending by conv2d_wgrad(pending=...)): that weight
    gradient's slab sum rides in this launch (acktr_conv2d_dgrad_carry_f32).
    gate_bits (int32 words written by conv2d_fwd(gate_mask=) of the layer that produced x_act): read instead of x_act."""
    OC, C, KH, KW = w.shape
    B, _, OH, OW = dy.shape
    H, W = (OH - 1) * stride + KH, (OW - 1) * stride + KW
    if out is None:
        out = torch.empty(B, C, H, W, dtype=f32, device=dy.device)
    assert out.shape == (B, C, H, W) and (x_act is None or x_act.shape == out.shape)
    pad = 0
    if padded_out is not None:
        pad = (padded_out.shape[-1] - W) // 2
        assert padded_out.shape == (B, C, H + 2 * pad, W + 2 * pad) and pad > 0
    assert not dy_prepadded or packed is not None
    L = _hip.lib()
    ws = packed if packed is not None else \
        workspace(dy.device, L.acktr_conv2d_dgrad_workspace_bytes(B, C, H, W, OC, KH, KW, stride), tag='dgrad')
    with _Timed('conv%ds%d_dgrad' % (KH, stride), 2.0 * dy.numel() * C * KH * KW):
        gate = _p(x_act, 'x_act')
        if gate_bits is not None:
            assert gate_bits.numel() * 4 >= L.acktr_conv2d_gate_mask_bytes(B, C, H, W)
            gate = _p(gate_bits, 'gate_bits', torch.int32)
        rc = L.acktr_conv2d_dgrad_carry_f32(_p(dy, 'dy'), _p(w, 'w'), gate, _p(out, 'dx'),
                                            B, C, H, W, OC, KH, KW, stride, _p(ws, 'workspace', torch.uint8), ws.numel(),
                                            (1 if packed is not None else 0) | (2 if dy_prepadded else 0)
                                            | (4 if gate_bits is not None else 0),
                                            _p(padded_out, 'dx_padded'), pad,
                                            ctypes.byref(carry) if (carry is not None and carry.dst) else None,
                                            _hip.cur_stream(dy.device))
    _hip.check(rc, 'acktr_conv2d_dgrad_carry_f32')
    return out


ACT = {None: 0, 'none': 0, 'relu': 1, 'tanh': 2}


def linear_fwd(x, w, bias, act=None, out=None):
    B, IN = x.shape
    OUT = w.shape[0]
    assert w.shape[1] == IN
    if out is None:
        out = torch.empty(B, OUT, dtype=f32, device=x.device)
    L = _hip.lib()
    nb = L.acktr_linear_fwd_workspace_bytes(B, IN, OUT)
    ws = workspace(x.device, nb) if nb else None
    with _Timed('linear%dx%d_fwd' % (IN, OUT), 2.0 * B * IN * OUT):
        rc = L.acktr_linear_fwd_f32(_p(x, 'x'), _p(w, 'w'), _p(bias, 'bias'), _p(out, 'y'), B, IN, OUT, ACT[act],
                                    _p(ws, 'workspace', torch.uint8), ws.numel() if ws is not None else 0,
                                    _hip.cur_stream(x.device))
    _hip.check(rc, 'acktr_linear_fwd_f32')
    return out


def linear_fwd_slabs(x, w):
    """x w^T as split-K slabs (no bias, no activation, no reduction): returns (workspace, nslabs, slab stride in floats).
    The slabs live in a scratch buffer of their own tag: valid until the next call on this device."""
    B, IN = x.shape
    OUT = w.shape[0]
    assert w.shape[1] == IN
    L = _hip.lib()
    ws = workspace(x.device, L.acktr_linear_fwd_slabs_workspace_bytes(B, IN, OUT), tag='fcslabs')
    ns = ctypes.c_int(0)
    with _Timed('linear%dx%d_fwd' % (IN, OUT), 2.0 * B * IN * OUT):
        rc = L.acktr_linear_fwd_slabs_f32(_p(x, 'x'), _p(w, 'w'), B, IN, OUT, _p(ws, 'workspace', torch.uint8), ws.numel(),
                                          ctypes.byref(ns), _hip.cur_stream(x.device))
    _hip.check(rc, 'acktr_linear_fwd_slabs_f32')
    return ws, ns.value, B * OUT


def linear_dgrad(dy, w, gate_src=None, gate=None, out=None, accumulate=False, padded_out=None, planes=None):
    """padded_out [B, C, OH+2p, OW+2p] with planes=(C, OH, OW): dx is also written there as zero-padded planes
    (interior only) -- the dY layout of the conv dgrad that follows an FC layer."""
    B, OUT = dy.shape
    IN = w.shape[1]
    assert w.shape[0] == OUT
    if out is None:
        assert not accumulate
        out = torch.empty(B, IN, dtype=f32, device=dy.device)
    C = OH = OW = pad = 0
    if padded_out is not None:
        C, OH, OW = planes
        pad = (padded_out.shape[-1] - OW) // 2
        assert C * OH * OW == IN and pad > 0 and padded_out.shape == (B, C, OH + 2 * pad, OW + 2 * pad)
    with _Timed('linear%dx%d_dgrad' % (IN, OUT), 2.0 * B * IN * OUT):
        rc = _hip.lib().acktr_linear_dgrad_ex_f32(_p(dy, 'dy'), _p(w, 'w'), _p(gate_src, 'gate_src'), ACT[gate],
                                                  _p(out, 'dx'), B, IN, OUT, 1 if accumulate else 0,
                                                  _p(padded_out, 'dx_padded'), C, OH, OW, pad,
                                                  _hip.cur_stream(dy.device))
    _hip.check(rc, 'acktr_linear_dgrad_ex_f32')
    return out


def linear_wgrad(dy, x, dw, db=None):
    B, OUT = dy.shape
    IN = x.shape[1]
    assert x.shape[0] == B and dw.numel() == OUT * IN and (db is None or db.numel() == OUT)
    L = _hip.lib()
    ws = workspace(dy.device, L.acktr_linear_wgrad_workspace_bytes(B, IN, OUT))
    with _Timed('linear%dx%d_wgrad' % (IN, OUT), 2.0 * B * IN * OUT):
        rc = L.acktr_linear_wgrad_f32(_p(dy, 'dy'), _p(x, 'x'), _p(dw, 'dw'), _p(db, 'db'), B, IN, OUT,
                                      _p(ws, 'workspace', torch.uint8), ws.numel(), _hip.cur_stream(dy.device))
    _hip.check(rc, 'acktr_linear_wgrad_f32')


def gemm(a, b, out=None, trans_a=False, trans_b=False, alpha=1.0, accumulate=False):
    """out (=|+=) alpha * op(a) @ op(b) for 2-D contiguous fp32 GPU tensors (op = transpose if trans_*)."""
    M, K = (a.shape[1], a.shape[0]) if trans_a else a.shape
    K2, N = (b.shape[1], b.shape[0]) if trans_b else b.shape
    assert K == K2, 'inner dimensions differ'
    if out is None:
        assert not accumulate
        out = torch.empty(M, N, dtype=f32, device=a.device)
    assert out.shape == (M, N) and out.is_contiguous()
    # A(m,k): a[m,k] -> (row stride lda, k stride 1); transposed: a[k,m] -> (row stride 1, k stride lda)
    a_sr, a_sk = (1, a.shape[1]) if trans_a else (a.shape[1], 1)
    # B(n,k) = op(b)[k,n]: b[k,n] -> (row stride 1, k stride ldb); transposed: b[n,k] -> (row stride ldb, k stride 1)
    b_sr, b_sk = (b.shape[1], 1) if trans_b else (1, b.shape[1])
    rc = _hip.lib().acktr_gemm_f32(_p(a, 'a'), a_sr, a_sk, _p(b, 'b'), b_sr, b_sk, _p(out, 'c'), N, M, N, K,
                                   float(alpha), 1 if accumulate else 0, _hip.cur_stream(a.device))
    _hip.check(rc, 'acktr_gemm_f32')
    return out


# ----------------------------------------------------------------------------------------------
# the gated recurrent core's operators (csrc/linear_act.hip, csrc/gated_scan.hip): bf16, fp16 or fp32 storage, fp32 arithmetic.
# Rows may be slices of wider ones (only the last axis has to be contiguous).  Scratch memory comes from torch's allocator
# per call, so calls on several streams, and graphs captured one after the other, do not share any.
# ----------------------------------------------------------------------------------------------
DTYPE_CODE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
LINEAR_ACT = {None: 0, 'none': 0, 'relu': 1, 'tanh': 2, 'silu': 3, 'gelu': 4}


class _on(object):
    """Kernels are launched on the operands' device, whichever device is current."""
    __slots__ = ('guard',)

    def __init__(self, index):
        self.guard = None if index == torch.cuda.current_device() else torch.cuda.device(index)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *a):
        if self.guard is not None:
            self.guard.__exit__(*a)
        return False


_current_device = getattr(torch._C, '_cuda_getDevice', torch.cuda.current_device)
_current_stream = getattr(torch._C, '_cuda_getCurrentRawStream', None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _launch(fn, index, what, work, *args):
    """fn(*args, stream) on device `index`, timed when the profiler is on."""
    if profiler is None and index == _current_device():
        rc = fn(*args, _current_stream(index))
    else:
        with _on(index), _Timed(what, work):
            rc = fn(*args, _current_stream(index))
    if rc:
        _hip.check(rc, 'acktr_' + what)


def _refuse(t, name, shape, dtype, index):
    """Says what is wrong with an operand that is not a GPU tensor of this shape, type and device with a contiguous last axis."""
    if not t.is_cuda:
        raise RuntimeError('%s must live on the MI355X device (got %s): this package has no CPU path' % (name, t.device))
    if t.get_device() != index:
        raise RuntimeError('%s is on %s, expected cuda:%d' % (name, t.device, index))
    if t.dtype != dtype:
        raise RuntimeError('%s must be %s (got %s)' % (name, dtype, t.dtype))
    if t.shape != shape:
        raise RuntimeError('%s must have shape %s (got %s)' % (name, tuple(shape), tuple(t.shape)))
    raise RuntimeError('%s: the last axis must be contiguous (strides %s)' % (name, tuple(t.stride())))


def _vec(t, name, n, dtype, index):
    if t.dtype is not dtype or t.get_device() != index or t.shape != (n,) or (n > 1 and t.stride(0) != 1):
        _refuse(t, name, (n,), dtype, index)
    return t.data_ptr()


def _rows(t, name, shape, dtype, index):
    """(pointer, row stride in elements) of a matrix whose rows may be slices of wider ones."""
    if t.dtype is not dtype or t.get_device() != index or t.shape != shape:
        _refuse(t, name, shape, dtype, index)
    ld, inner = t.stride()
    if inner != 1 and shape[1] > 1:
        _refuse(t, name, shape, dtype, index)
    return t.data_ptr(), (ld if shape[0] > 1 else max(shape[1], 1))


def _dense(t, name, shape, dtype, index):
    if t.dtype is not dtype or t.get_device() != index or t.shape != shape:
        _refuse(t, name, shape, dtype, index)
    if not t.is_contiguous():
        raise RuntimeError('%s must be contiguous' % name)
    return t.data_ptr()


def _dtype_code(t, name):
    code = DTYPE_CODE.get(getattr(t, 'dtype', None))
    if code is None:
        raise RuntimeError('%s must be a bfloat16, float16 or float32 tensor (got %s)' % (name, getattr(t, 'dtype', type(t))))
    if not t.is_cuda:
        raise RuntimeError('%s must live on the MI355X device (got %s): this package has no CPU path' % (name, t.device))
    return code


def _act_code(act):
    code = LINEAR_ACT.get(act)
    if code is None:
        raise RuntimeError('unknown activation %r (one of none, relu, tanh, silu, gelu)' % (act,))
    return code


def _reach(t):
    """[first byte, last byte + 1) of a tensor"""
    if t is None:
        return 0, 0
    p = t.data_ptr()
    if t.is_contiguous():
        return p, p + t.nbytes
    if t.numel() == 0:
        return 0, 0
    return p, p + (1 + sum([(n - 1) * s for n, s in zip(t.shape, t.stride())])) * t.element_size()


def _apart(out, name, others, what):
    """`out` (to be written; its elements must not share memory) has no element in common with any of `others`."""
    if not out.is_contiguous():
        reach = 1
        for s, n in sorted((s, n) for n, s in zip(out.shape, out.stride()) if n > 1):
            if s < reach:
                raise RuntimeError('%s: %s has elements that share memory (strides %s)' % (what, name, tuple(out.stride())))
            reach += s * (n - 1)
    a0, a1 = _reach(out)
    for t in others:
        if t is None or t.data_ptr() >= a1:
            continue
        b0, b1 = _reach(t)
        if a0 < b1 and b0 < a1 and not _side_by_side(out, a0, t, b0):
            raise RuntimeError('%s: %s overlaps another operand' % (what, name))


def _side_by_side(a, a0, b, b0):
    """Column slices of the same rows: their spans cross, their elements do not."""
    e = a.element_size()
    if a.dim() != b.dim() or a.dim() < 2 or a.stride() != b.stride() or b.element_size() != e or (b0 - a0) % e:
        return False
    steps = [s for n, s in zip(a.shape[:-1], a.stride()[:-1]) if n > 1]
    if not steps or min(steps) <= 0 or any(s % min(steps) for s in steps):
        return False
    d = (b0 - a0) // e % min(steps)
    return d >= a.shape[-1] and d + b.shape[-1] <= min(steps)


def _scratch(nbytes, like, what):
    if nbytes < 0:
        _hip.check(-1, what)
    return like.new_empty(nbytes, dtype=torch.uint8)


# A kernel writes through a pointer, which autograd does not see: every tensor of the caller's that a call wrote is marked as changed, so
# that a backward pass that still needs its old values raises instead of using the new ones.
_written = torch.autograd.graph.increment_version


def linear_act_fwd(x, w, bias=None, act=None, residual=None, out=None, pre=None):
    """out = act(x w^T + bias) + residual; x [M, K], w [N, K], bias [N], residual / out / pre [M, N], all of one type (bf16, fp16 or
    fp32), sums in fp32, rounded once.  act: None, 'relu', 'tanh', 'silu' or 'gelu'.  pre [M, N]: receives
    what linear_act_bwd needs of the pre-activations (the activation's slopes, encoded).  out may be `residual` itself."""
    code, act = _dtype_code(x, 'x'), _act_code(act)
    mk, nk = x.shape, w.shape
    if len(mk) != 2 or len(nk) != 2 or mk[1] != nk[1] or mk[1] < 1 or nk[0] < 1:
        raise RuntimeError('linear_act_fwd: x [M, K] and w [N, K] expected, got %s and %s' % (tuple(mk), tuple(nk)))
    (M, K), N, dt, at = mk, nk[0], x.dtype, x.get_device()
    mn = (M, N)
    given = out is not None
    if not given:
        out = x.new_empty(mn)
    px, ldx = _rows(x, 'x', mk, dt, at)
    pw, ldw = _rows(w, 'w', nk, dt, at)
    py, ldy = _rows(out, 'out', mn, dt, at)
    pb = _vec(bias, 'bias', N, dt, at) if bias is not None else None
    pr, ldr = _rows(residual, 'residual', mn, dt, at) if residual is not None else (None, 0)
    pz, ldz = None, 0
    if pre is not None:
        pz, ldz = _rows(pre, 'pre', mn, dt, at)
        _apart(pre, 'pre', (x, w, bias, residual, out if given else None), 'linear_act_fwd')
    if given:
        _apart(out, 'out', (x, w, bias, None if pr == py and ldr == ldy else residual), 'linear_act_fwd')
    L = _hip.lib()
    nb = L.acktr_linear_act_fwd_workspace_bytes(px, ldx, pw, ldw, M, N, K, code)
    ws = _scratch(nb, x, 'acktr_linear_act_fwd') if nb else None
    _launch(L.acktr_linear_act_fwd, at, 'linear_act_fwd', 2.0 * M * N * K, px, ldx, pw, ldw, pb, pr, ldr, py, ldy, pz, ldz, M, N, K, code,
            act, ws.data_ptr() if nb else None, nb)
    if pre is not None:
        _written(pre)
    if given:
        _written(out)
    return out


def linear_act_bwd(dy, x, w, pre=None, act=None, dx=None, dw=None, db=None, need_dx=True, need_dw=True, need_db=True, dx_add=None):
    """(dx, dw, db) of linear_act_fwd for dy [M, N] = the derivative by its output (the residual's gradient is dy itself).
    pre: what the forward pass left there (not needed without an activation).  dx_add [M, K]: added to dx
    before it is rounded (what reaches x by another way, a residual's gradient).  Gradients that are not needed are None."""
    code, act = _dtype_code(dy, 'dy'), _act_code(act)
    if dy.dim() != 2 or x.dim() != 2 or w.dim() != 2 or x.shape[0] != dy.shape[0] or tuple(w.shape) != (dy.shape[1], x.shape[1]):
        raise RuntimeError('linear_act_bwd: dy [M, N], x [M, K] and w [N, K] expected, got %s, %s and %s'
                           % (tuple(dy.shape), tuple(x.shape), tuple(w.shape)))
    (M, N), K, dt, at = dy.shape, x.shape[1], dy.dtype, dy.get_device()
    if act and pre is None:
        raise RuntimeError("linear_act_bwd: an activation's gradient needs `pre` of the forward pass")
    if not act:
        pre = None
    given = [t for t, need in ((dx, need_dx), (dw, need_dw), (db, need_db)) if need and t is not None]
    pg, ldg = _rows(dy, 'dy', (M, N), dt, at)
    px, ldx = _rows(x, 'x', (M, K), dt, at)
    pw, ldw = _rows(w, 'w', (N, K), dt, at)
    pz, ldz = _rows(pre, 'pre', (M, N), dt, at) if pre is not None else (None, 0)
    qx = qw = qb = pa = None
    ldq = lda = 0
    if dx_add is not None:
        pa, lda = _rows(dx_add, 'dx_add', (M, K), dt, at)
    if need_dx:
        dx = dy.new_empty((M, K)) if dx is None else dx
        qx, ldq = _rows(dx, 'dx', (M, K), dt, at)
    if need_dw:
        dw = dy.new_empty((N, K)) if dw is None else dw
        qw = _dense(dw, 'dw', (N, K), dt, at)
    if need_db:
        db = dy.new_empty(N) if db is None else db
        qb = _vec(db, 'db', N, dt, at)
    for i, a in enumerate(given):
        _apart(a, 'a gradient', (dy, x, w, pre, None if a is dx and qx == pa and ldq == lda else dx_add) + tuple(given[:i]), 'linear_act_bwd')
    L = _hip.lib()
    nb = L.acktr_linear_act_bwd_workspace_bytes(pg, ldg, px, ldx, pw, ldw, pz, ldz, need_dx, need_dw, need_db, M, N, K, code, act)
    ws = _scratch(nb, dy, 'acktr_linear_act_bwd') if nb else None
    _launch(L.acktr_linear_act_bwd, at, 'linear_act_bwd', 2.0 * M * N * K * (bool(need_dx) + bool(need_dw)), pg, ldg, px, ldx, pw, ldw, pz, ldz,
            pa, lda, qx, ldq, qw, qb, M, N, K, code, act, ws.data_ptr() if nb else None, nb)
    if given:
        _written(given)
    return dx if need_dx else None, dw if need_dw else None, db if need_db else None


def _steps(t, name, shape, dtype, index):
    """(pointer, stride over steps, stride over sequences) of a [T, N, H] operand; axes of one element take a packed stride."""
    if t.dtype is not dtype or t.get_device() != index or t.shape != shape:
        _refuse(t, name, shape, dtype, index)
    st, sn, inner = t.stride()
    T, N, H = shape
    if inner != 1 and H > 1:
        _refuse(t, name, shape, dtype, index)
    return t.data_ptr(), (st if T > 1 else N * H), (sn if N > 1 else H)


def _span3(q, shape, e):
    """[first byte, last byte + 1) of a [T, N, H] operand (pointer, strides) of e-byte elements"""
    p, st, sn = q
    T, N, H = shape
    return p, (p + ((T - 1) * st + (N - 1) * sn + H) * e if T and N else p)


def _steps_apart(t, name, q, shape, e, spans, others, what):
    """_apart for a [T, N, H] operand that is written: by its strides and the others' spans where those settle it"""
    _, st, sn = q
    T, N, H = shape
    lo, hi = _span3(q, shape, e)
    if (sn >= H and st >= (N - 1) * sn + H) or (st >= H and sn >= (T - 1) * st + H):
        for a, b in spans:
            if a < hi and lo < b:
                break
        else:
            return
    _apart(t, name, others, what)


def _masks(masks, shape, index):
    """[T, N] fp32 or the rollout's [T, N, 1]"""
    if masks is None:
        return None
    if masks.dim() == len(shape) + 1 and masks.shape[-1] == 1:
        masks = masks.squeeze(-1)
    return _dense(masks, 'masks', shape, f32, index)


_interval = None


def _scan_interval():
    global _interval
    if _interval is None:
        _interval = _hip.lib().acktr_gated_scan_save_interval()
    return _interval


def gated_scan_fwd(gate, value, h0=None, masks=None, out=None, save=False):
    """(out, last, saved) of the gated linear recurrence h_t = f_t (m_t h_{t-1}) + (1 - f_t) value_t, f = sigmoid(gate).
    gate, value, out [T, N, H] (one type; any strides over T and N: halves of one projection, batch-first views); h0 [N, H] fp32 or
    None (zeros); masks [T, N] or [T, N, 1] fp32 or None (ones): where it is 0 nothing before counts.  last [N, H] fp32: the final
    state.  save=True: the states that gated_scan_bwd starts from, else None."""
    code = _dtype_code(gate, 'gate')
    if gate.dim() != 3 or gate.shape[2] < 1:
        raise RuntimeError('gated_scan_fwd: gate [T, N, H] expected, got %s' % (tuple(gate.shape),))
    shape, dt, at = gate.shape, gate.dtype, gate.get_device()
    T, N, H = shape
    given = out is not None
    if not given:
        out = gate.new_empty(shape)
    pg, pv, po = _steps(gate, 'gate', shape, dt, at), _steps(value, 'value', shape, dt, at), _steps(out, 'out', shape, dt, at)
    ph = _dense(h0, 'h0', (N, H), f32, at) if h0 is not None else None
    pm = _masks(masks, (T, N), at)
    if given:
        e, c = out.element_size(), 4 * N * H
        spans = (_span3(pg, shape, e), _span3(pv, shape, e), (ph or 0, ph + c if ph else 0), (pm or 0, pm + 4 * T * N if pm else 0))
        _steps_apart(out, 'out', po, shape, e, spans, (gate, value, h0, masks), 'gated_scan_fwd')
    L = _hip.lib()
    last = gate.new_empty((N, H), dtype=f32)
    saved = gate.new_empty((-(-T // _scan_interval()), N, H), dtype=f32) if save else None
    nb = L.acktr_gated_scan_workspace_bytes(T, N, H, code)
    ws = _scratch(nb, gate, 'acktr_gated_scan_fwd') if nb else None
    _launch(L.acktr_gated_scan_fwd, at, 'gated_scan_fwd', 10.0 * T * N * H, *pg, *pv, ph, pm, *po, last.data_ptr(),
            saved.data_ptr() if save else None, T, N, H, code, ws.data_ptr() if nb else None, nb)
    if given:
        _written(out)
    return out, last, saved


def gated_scan_bwd(dout, gate, value, h0=None, masks=None, saved=None, dlast=None, dgate=None, dvalue=None, need_dh0=True):
    """(dgate, dvalue, dh0) for dout [T, N, H] = the derivative by the states and dlast [N, H] fp32 (or None) by the final one;
    the other operands are those of gated_scan_fwd(save=True) and what it saved."""
    code = _dtype_code(gate, 'gate')
    if gate.dim() != 3 or gate.shape[2] < 1:
        raise RuntimeError('gated_scan_bwd: gate [T, N, H] expected, got %s' % (tuple(gate.shape),))
    shape, dt, at = gate.shape, gate.dtype, gate.get_device()
    T, N, H = shape
    given = [t for t in (dgate, dvalue) if t is not None]
    dgate = gate.new_empty(shape) if dgate is None else dgate
    dvalue = gate.new_empty(shape) if dvalue is None else dvalue
    pd, pg, pv = _steps(dout, 'dout', shape, dt, at), _steps(gate, 'gate', shape, dt, at), _steps(value, 'value', shape, dt, at)
    qg, qv = _steps(dgate, 'dgate', shape, dt, at), _steps(dvalue, 'dvalue', shape, dt, at)
    L = _hip.lib()
    every = _scan_interval()
    ph = _dense(h0, 'h0', (N, H), f32, at) if h0 is not None else None
    pm = _masks(masks, (T, N), at)
    ps = _dense(saved, 'saved', (-(-T // every), N, H), f32, at) if saved is not None and T else None
    pl = _dense(dlast, 'dlast', (N, H), f32, at) if dlast is not None else None
    if T > every and saved is None:
        raise RuntimeError('gated_scan_bwd: more than %d steps need what gated_scan_fwd(save=True) saved' % every)
    if given:
        e, c = gate.element_size(), 4 * N * H
        spans = [_span3(pd, shape, e), _span3(pg, shape, e), _span3(pv, shape, e), (ph or 0, ph + c if ph else 0), (pm or 0, pm + 4 * T * N if pm else 0),
                 (ps or 0, ps + -(-T // every) * c if ps else 0), (pl or 0, pl + c if pl else 0)]
        reads = (dout, gate, value, h0, masks, saved, dlast)
        for a in given:
            _steps_apart(a, 'a gradient', qg if a is dgate else qv, shape, e, spans, reads, 'gated_scan_bwd')
        if len(given) == 2:
            _apart(dgate, 'dgate', (dvalue,), 'gated_scan_bwd')
    dh0 = gate.new_empty((N, H), dtype=f32) if need_dh0 else None
    nb = L.acktr_gated_scan_workspace_bytes(T, N, H, code)
    ws = _scratch(nb, gate, 'acktr_gated_scan_bwd') if nb else None
    _launch(L.acktr_gated_scan_bwd, at, 'gated_scan_bwd', 20.0 * T * N * H, *pd, *pg, *pv, ph, pm, ps, pl, *qg, *qv,
            dh0.data_ptr() if need_dh0 else None, T, N, H, code, ws.data_ptr() if nb else None, nb)
    if given:
        _written(given)
    return dgate, dvalue, dh0


def gated_scan_step(gate, value, state, masks=None, out=None):
    """One step of the recurrence: state [N, H] fp32 is updated IN PLACE, the result is returned rounded to gate's type.
    gate, value, out [N, H]; masks [N] or [N, 1] fp32 or None."""
    code = _dtype_code(gate, 'gate')
    if gate.dim() != 2 or gate.shape[1] < 1:
        raise RuntimeError('gated_scan_step: gate [N, H] expected, got %s' % (tuple(gate.shape),))
    shape, dt, at = gate.shape, gate.dtype, gate.get_device()
    N, H = shape
    given = out is not None
    if not given:
        out = gate.new_empty(shape)
    (pg, gn), (pv, vn), (po, on) = _rows(gate, 'gate', shape, dt, at), _rows(value, 'value', shape, dt, at), _rows(out, 'out', shape, dt, at)
    ps = _dense(state, 'state', shape, f32, at)
    pm = _masks(masks, (N,), at)
    if given:
        _apart(out, 'out', (gate, value, state, masks), 'gated_scan_step')
    lo, hi = ps, ps + 4 * N * H
    # (a row that all sequences share has a stride of 0, and still H values)
    if lo <= pg < hi or lo <= pv < hi or pg <= lo < pg + max(gn, H) * N * 4 or pv <= lo < pv + max(vn, H) * N * 4 or (pm and lo - 4 * N < pm < hi):
        _apart(state, 'state', (gate, value, masks), 'gated_scan_step')
    _launch(_hip.lib().acktr_gated_scan_step, at, 'gated_scan_step', 10.0 * N * H, pg, gn, pv, vn, ps, pm, po, on, N, H, code)
    _written((state, out) if given else state)
    return out


def gated_core_step(x, w_in, b_in, w_out, b_out, state, masks=None, state_out=None):
    """(y, state_out) of one step of the gated core (gated.GatedCore): x [N, I], w_in [2H, I], w_out [H, H] of one type, biases [2H] and
    [H] or None, state [N, H] fp32, masks [N] or [N, 1] fp32 or None.  state_out: receives the new state and may be `state` itself
    (default: a new tensor).  The same results as linear_act_fwd, gated_scan_step and linear_act_fwd, in one call."""
    code = _dtype_code(x, 'x')
    if x.dim() != 2 or w_in.dim() != 2 or w_in.shape[1] != x.shape[1] or x.shape[1] < 1 or w_in.shape[0] < 2 or w_in.shape[0] % 2:
        raise RuntimeError('gated_core_step: x [N, I] and w_in [2H, I] expected, got %s and %s' % (tuple(x.shape), tuple(w_in.shape)))
    (N, I), H, dt, at = x.shape, w_in.shape[0] // 2, x.dtype, x.get_device()
    px, ldx = _rows(x, 'x', x.shape, dt, at)
    pi, po = _dense(w_in, 'w_in', (2 * H, I), dt, at), _dense(w_out, 'w_out', (H, H), dt, at)
    bi = _vec(b_in, 'b_in', 2 * H, dt, at) if b_in is not None else None
    bo = _vec(b_out, 'b_out', H, dt, at) if b_out is not None else None
    ps = _dense(state, 'state', (N, H), f32, at)
    pm = _masks(masks, (N,), at)
    given = state_out is not None
    if not given:
        state_out = state.new_empty((N, H))
    else:
        pq = _dense(state_out, 'state_out', (N, H), f32, at)
        _apart(state_out, 'state_out', (x, w_in, b_in, w_out, b_out, masks, None if pq == ps else state), 'gated_core_step')
    y = x.new_empty((N, H))
    L = _hip.lib()
    nb = L.acktr_gated_core_step_workspace_bytes(px, ldx, pi, po, N, I, H, code)
    ws = _scratch(nb, x, 'acktr_gated_core_step')
    _launch(L.acktr_gated_core_step, at, 'gated_core_step', 4.0 * N * H * I + 2.0 * N * H * H, px, ldx, pi, bi, po, bo, ps, state_out.data_ptr(),
            pm, y.data_ptr(), H, N, I, H, code, ws.data_ptr(), nb)
    if given:
        _written(state_out)
    return y, state_out
