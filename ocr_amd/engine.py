"""Thin host layer over the C ABI: torch tensors in, torch tensors out.

PyTorch is used for device memory and streams only; every computation below happens inside
libocrhip.so.  One `HipContext` per (device, host thread).
"""
import ctypes
from typing import NamedTuple

import numpy as np
import torch

from . import _lib
from ._lib import F32, BF16, U8, MERGE_UNION, MERGE_AVERAGE, MERGE_WEIGHTED, TensorDesc, check

# types of the operands and results of the 8-bit products and the distillation
_VALUES = {torch.float32: F32, torch.bfloat16: BF16}
_MERGE = {'union': MERGE_UNION, 'average': MERGE_AVERAGE, 'weighted': MERGE_WEIGHTED}


_BYTES = (torch.float8_e4m3fn, torch.uint8)
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, '_cuda_getCurrentRawStream') else \
    lambda index: torch.cuda.current_stream(index).cuda_stream


def _address(t):
    return None if t is None else t.data_ptr()


def _ptr(t):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else None


def _uniform_stride(t):
    """Element stride of a tensor whose elements lie at base + k * stride, k = 0..numel-1 in row-major order (a
    contiguous tensor: 1; `m[..., 0]` of a contiguous (h,w,6) map: 6); None when there is no such stride."""
    if t.numel() <= 1:
        return 1
    dims = [(n, st) for n, st in zip(t.shape, t.stride()) if n > 1]
    step = dims[-1][1]
    expect = step
    for n, st in reversed(dims):
        if st != expect:
            return None
        expect = st * n
    return step if step >= 1 else None


def _stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _descs(state_dict):
    """state dict (torch tensors or arrays) -> (ctypes array of TensorDesc, keep-alive list)."""
    keep, items = [], []
    for name, value in state_dict.items():
        if name.startswith('module.'):
            name = name[len('module.'):]
        if name.endswith('num_batches_tracked'):
            continue
        arr = value.detach().cpu().numpy() if isinstance(value, torch.Tensor) else np.asarray(value)
        arr = np.ascontiguousarray(arr, dtype=np.float32)
        if arr.ndim > 4:
            continue
        bname = name.encode('utf-8')
        keep.append((arr, bname))
        d = TensorDesc()
        d.name = bname
        d.data = arr.ctypes.data
        d.ndim = arr.ndim
        for i in range(arr.ndim):
            d.shape[i] = arr.shape[i]
        items.append(d)
    array = (TensorDesc * len(items))(*items)
    return array, keep


class Fp8Matrix(NamedTuple):
    """A matrix in 8-bit floating point with a power-of-two scale per block of `block_rows` (1 or 128) rows x 128 columns:
    element (r, c) = q[r, c] * 2 ** (scale[c // 128, r // block_rows] - 127).  What `HipContext.quantize_fp8` returns and
    `gemm_fp8` / `linear_fp8` take."""
    q: torch.Tensor            # (rows, columns rounded up to a multiple of 128) float8_e4m3fn, zero behind the last column
    scale: torch.Tensor        # (ceil(cols / 128), number of row blocks rounded up to a multiple of 16) uint8
    rows: int
    cols: int
    block_rows: int


class HipContext:
    """Owns one ocrhip handle (weights + workspaces) on one GPU."""

    def __init__(self, device=0):
        if not torch.cuda.is_available():
            raise RuntimeError('ocr_amd needs a ROCm GPU (torch.cuda.is_available() is False)')
        self.lib = _lib.load()
        self.device = torch.device('cuda', device)
        h = ctypes.c_void_p()
        check(self.lib.ocrhip_create(int(device), ctypes.byref(h)))
        self._h = h
        self.east_loaded = False
        self.crnn_loaded = False
        self.options = {}              # what set_option was last called with, per name

    def close(self):
        if getattr(self, '_h', None):
            self.lib.ocrhip_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    # ------------------------------------------------------------------ stage timers
    def profile_enable(self, enable=True):
        check(self.lib.ocrhip_profile_enable(self._h, 1 if enable else 0))

    def profile_only(self, name=None):
        """Times only the launches recorded under `name` (None: all of them again)."""
        check(self.lib.ocrhip_profile_only(self._h, name.encode() if name else None))

    def profile_collect(self, cap=64):
        """-> list of dict(name, launches, total_ms, flops, bytes) sorted by total time (synchronises)."""
        arr = (_lib.KernelStat * cap)()
        n = ctypes.c_int(0)
        check(self.lib.ocrhip_profile_collect(self._h, arr, cap, ctypes.byref(n)))
        return [{'name': arr[i].name.decode(), 'launches': arr[i].launches, 'total_ms': arr[i].total_ms,
                 'flops': arr[i].flops, 'bytes': arr[i].bytes} for i in range(min(cap, n.value))]

    # ------------------------------------------------------------------ EAST
    def east_load_weights(self, state_dict):
        arr, keep = _descs(state_dict)
        check(self.lib.ocrhip_east_load_weights(self._h, arr, len(arr)))
        self.east_loaded = True

    def set_option(self, name, value):
        """'conv3x3_winograd': 2 (default) Winograd F(4x4,3x3) where the map fills its tiles and F(2x2,3x3) elsewhere,
        1 F(2x2,3x3) for all wide 3x3 convolutions, 0 direct implicit GEMM.
        'lstm_persistent': 2 (default) one persistent launch per BiLSTM layer (independent waves on blocks of 16
        sequences for large batches, workgroup-wide passes otherwise), 1 passes always, 3 independent waves always,
        0 one launch per time step.
        'lstm16_units': 64 (default) or 32 hidden units per workgroup of the bfloat16 recurrence.
        'crnn_side_streams': 1 (default) many small width groups of a packed batch run on side streams, 0 on one stream.
        'fuse_mean_rows': 1 (default) the mean over the feature rows in the last convolution's epilogue, 0 a kernel of its own.
        'bf16_fuse_first': 1 (default) the bfloat16 detector's first two layers in one launch, 0 two launches.
        'wino4_split': 0 (default) every F(4x4,3x3) layer fused, 1 layers with >= 512 input channels as transform kernel +
        multiply kernel.
        'flat_gemm': 1 (default) Dense layers / LSTM input projections / 2x2 convolutions on the 256 x 128 flat GEMM,
        0 on the implicit-GEMM convolution kernel.
        'fp8_dense': 1 the dense layers of the bfloat16 recogniser as 8-bit block-scaled products (logits within 0.2 of the
        bfloat16 ones in norm; switching it on quantises their weights, which takes 5 ms), 0 (default) on bfloat16 operands."""
        check(self.lib.ocrhip_set_option(self._h, name.encode(), int(value)))
        self.options[name] = int(value)

    def image_resize_norm(self, images, out_h, out_w):
        """images: (B,H,W,3) uint8 raw or float32 in [0,1], on the GPU -> (B,out_h,out_w,3) float32 normalised
        network input (`/255` for uint8, antialiased bilinear stretch, `(x-0.5)/0.5`)."""
        assert images.is_cuda and images.dim() == 4 and images.shape[3] == 3 and images.is_contiguous()
        if images.dtype == torch.uint8:
            in_dtype = U8
        elif images.dtype == torch.float32:
            in_dtype = F32
        else:
            raise ValueError('image_resize_norm: images must be uint8 or float32')
        B, H, W, _ = images.shape
        out = torch.empty((B, int(out_h), int(out_w), 3), dtype=torch.float32, device=images.device)
        check(self.lib.ocrhip_image_resize_norm(self._h, _ptr(images), in_dtype, B, H, W, int(out_h), int(out_w),
                                                _ptr(out), _stream()))
        return out

    def dice_coeff(self, x, y):
        """Dice coefficient 2*sum(x*y) / (sum(x)+sum(y)) of two float32 GPU tensors of one shape (0 when both are all
        zero) -> float32 GPU scalar.  Views that step over whole elements (`maps[..., 0]` of a contiguous map) are
        walked in place."""
        assert x.is_cuda and y.is_cuda and x.dtype == torch.float32 and y.dtype == torch.float32
        if tuple(x.shape) != tuple(y.shape):
            raise ValueError('dice_coeff: shapes differ: {} vs {}'.format(tuple(x.shape), tuple(y.shape)))
        stride = _uniform_stride(x)
        if stride is None or _uniform_stride(y) != stride:
            x, y, stride = x.contiguous(), y.contiguous(), 1
        out = torch.empty((1,), dtype=torch.float32, device=x.device)
        check(self.lib.ocrhip_dice_coeff(self._h, _ptr(x), _ptr(y), x.numel(), stride, _ptr(out), _stream()))
        return out[0]

    def east_forward(self, images, compute_dtype=F32):
        """images: (B,H,W,3) uint8 raw or float32 normalised, on the GPU -> (B,H/4,W/4,6) float32."""
        assert images.is_cuda and images.dim() == 4 and images.shape[3] == 3 and images.is_contiguous()
        if images.dtype == torch.uint8:
            in_dtype = U8
        elif images.dtype == torch.float32:
            in_dtype = F32
        else:
            raise ValueError('east_forward: images must be uint8 or float32')
        B, H, W, _ = images.shape
        maps = torch.empty((B, H // 4, W // 4, 6), dtype=torch.float32, device=images.device)
        check(self.lib.ocrhip_east_forward(self._h, _ptr(images), B, H, W, in_dtype, compute_dtype, _ptr(maps), _stream()))
        return maps

    def _activation(self, fn, name):
        shape = (ctypes.c_int64 * 4)()
        check(fn(self._h, name.encode(), None, 0, shape))
        out = np.empty(tuple(int(s) for s in shape), dtype=np.float32)
        check(fn(self._h, name.encode(), out.ctypes.data, out.size, shape))
        return out

    def east_activation(self, name):
        return self._activation(self.lib.ocrhip_east_get_activation, name)

    def east_decode(self, maps, input_hw, threshold=0.35, cap=None, with_polys=False, with_pix=False):
        """maps (B,mh,mw,6) -> dict(xyxy (B,cap,4), scores (B,cap), counts (B,), [polys (B,cap,4,2)], [pix])."""
        assert maps.is_cuda and maps.dtype == torch.float32 and maps.is_contiguous()
        B, mh, mw, _ = maps.shape
        if cap is None:
            cap = mh * mw
        dev = maps.device
        out = {
            'xyxy': torch.empty((B, cap, 4), dtype=torch.float32, device=dev),
            'scores': torch.empty((B, cap), dtype=torch.float32, device=dev),
            'counts': torch.empty((B,), dtype=torch.int32, device=dev),
        }
        polys = torch.empty((B, cap, 4, 2), dtype=torch.float32, device=dev) if with_polys else None
        pix = torch.empty((B, cap), dtype=torch.int32, device=dev) if with_pix else None
        check(self.lib.ocrhip_east_decode(self._h, _ptr(maps), B, mh, mw, int(input_hw[0]), int(input_hw[1]),
                                          float(threshold), int(cap), _ptr(out['xyxy']), _ptr(polys),
                                          _ptr(out['scores']), _ptr(pix), _ptr(out['counts']), _stream()))
        if with_polys:
            out['polys'] = polys
        if with_pix:
            out['pix'] = pix
        return out

    def lanms(self, xyxy, scores, counts, merge_threshold=0.3, nms_threshold=0.25, merge_method='union',
              max_iter=0, max_out=0, full=False):
        """xyxy (B,cap,4), scores (B,cap) or None, counts (B,) int32 ->
        dict(boxes (B,cap,4) rank order, scores, src, counts, n_iter, [merged, keep in input order])."""
        assert xyxy.is_cuda and xyxy.dtype == torch.float32 and xyxy.is_contiguous()
        B, cap, _ = xyxy.shape
        dev = xyxy.device
        out = {
            'boxes': torch.empty((B, cap, 4), dtype=torch.float32, device=dev),
            'scores': torch.empty((B, cap), dtype=torch.float32, device=dev),
            'src': torch.empty((B, cap), dtype=torch.int32, device=dev),
            'counts': torch.empty((B,), dtype=torch.int32, device=dev),
            'n_iter': torch.empty((B,), dtype=torch.int32, device=dev),
        }
        merged = torch.empty((B, cap, 4), dtype=torch.float32, device=dev) if full else None
        keep = torch.empty((B, cap), dtype=torch.uint8, device=dev) if full else None
        check(self.lib.ocrhip_lanms(self._h, _ptr(xyxy), _ptr(scores), _ptr(counts), B, cap, float(merge_threshold),
                                    float(nms_threshold), _MERGE[merge_method], int(max_iter or 0), int(max_out or 0),
                                    _ptr(merged), _ptr(keep), _ptr(out['boxes']), _ptr(out['scores']), _ptr(out['src']),
                                    _ptr(out['counts']), _ptr(out['n_iter']), _stream()))
        if full:
            out['merged'], out['keep'] = merged, keep
        return out

    # ------------------------------------------------------------------ crop / pack
    def crop_resize_pack(self, images, rects, box_img, inter_hw, out_w, dst_off, total_elems, out_h=64,
                         out_dtype=torch.float32):
        """images (B,H,W,3) uint8; rects (n,4) int32; box_img (n,) int32; inter_hw (n,2) int32; out_w (n,) int32;
        dst_off (n,) int64 -> flat packed buffer of `total_elems` elements."""
        assert images.is_cuda and images.dtype == torch.uint8 and images.is_contiguous()
        B, H, W, _ = images.shape
        n = int(rects.shape[0])
        packed = torch.empty((int(total_elems),), dtype=out_dtype, device=images.device)
        code = F32 if out_dtype == torch.float32 else BF16
        check(self.lib.ocrhip_crop_resize_pack(self._h, _ptr(images), B, H, W, _ptr(rects), _ptr(box_img), _ptr(inter_hw),
                                               _ptr(out_w), _ptr(dst_off), n, int(out_h), _ptr(packed), code, _stream()))
        return packed

    def crop_rotated_pack(self, images, geom, box_img, inter_hw, out_w, dst_off, total_elems, out_h=64,
                          out_dtype=torch.float32):
        """`crop_resize_pack` for oriented rectangles: geom (n,8) float32 = origin x, y, step along the text (x, y),
        step across the text (x, y), crop width, crop height (see `utils.image_sizes.plan_crops_rotated`)."""
        assert images.is_cuda and images.dtype == torch.uint8 and images.is_contiguous()
        assert geom.dtype == torch.float32 and geom.is_contiguous() and geom.shape[1] == 8
        B, H, W, _ = images.shape
        n = int(geom.shape[0])
        packed = torch.empty((int(total_elems),), dtype=out_dtype, device=images.device)
        code = F32 if out_dtype == torch.float32 else BF16
        check(self.lib.ocrhip_crop_rotated_pack(self._h, _ptr(images), B, H, W, _ptr(geom), _ptr(box_img), _ptr(inter_hw),
                                                _ptr(out_w), _ptr(dst_off), n, int(out_h), _ptr(packed), code, _stream()))
        return packed

    def rotated_nms(self, polys, scores, counts, iou_threshold, max_out=2048):
        """Greedy NMS with rotated IoU on decoded quadrilaterals: polys (B,cap,4,2) or (B,cap,8) float32, scores
        (B,cap), counts (B,) int32, all on the GPU -> dict(polys (B,max_out,4,2), scores, index (B,max_out) int32,
        counts (B,) int32), kept quadrilaterals in descending score order."""
        assert polys.is_cuda and polys.dtype == torch.float32 and polys.is_contiguous()
        assert scores.dtype == torch.float32 and scores.is_contiguous() and counts.dtype == torch.int32
        B, cap = int(scores.shape[0]), int(scores.shape[1])
        assert polys.numel() == B * cap * 8
        dev = polys.device
        out = {'polys': torch.zeros((B, int(max_out), 4, 2), dtype=torch.float32, device=dev),
               'scores': torch.zeros((B, int(max_out)), dtype=torch.float32, device=dev),
               'index': torch.full((B, int(max_out)), -1, dtype=torch.int32, device=dev),
               'counts': torch.zeros((B,), dtype=torch.int32, device=dev)}
        check(self.lib.ocrhip_rotated_nms(self._h, _ptr(polys), _ptr(scores), _ptr(counts), B, cap, float(iou_threshold),
                                          int(max_out), _ptr(out['polys']), _ptr(out['scores']), _ptr(out['index']),
                                          _ptr(out['counts']), _stream()))
        return out

    # ------------------------------------------------------------------ CRNN
    def crnn_load_weights(self, state_dict):
        arr, keep = _descs(state_dict)
        check(self.lib.ocrhip_crnn_load_weights(self._h, arr, len(arr)))
        self.crnn_loaded = True

    @property
    def vocab_size(self):
        return int(self.lib.ocrhip_crnn_vocab_size(self._h))

    def seq_len(self, wpad):
        """Time steps of the loaded recogniser for padded crop width(s) `wpad` (VGG: w/4 - 1, ResNet: w/4 + 1)."""
        delta = int(self.lib.ocrhip_crnn_seq_len(self._h, 8)) - 2
        if delta not in (-1, 1):
            raise RuntimeError('seq_len: recogniser weights are not loaded')
        return np.asarray(wpad) // 4 + delta

    def crnn_forward(self, crops, want_logits=True, want_tokens=False, compute_dtype=F32):
        """crops (n,64,Wpad,1) or (n,64,Wpad) float32 -> dict(logits (n,T,V), tokens (n,T), scores (n,))."""
        assert crops.is_cuda and crops.dtype == torch.float32 and crops.is_contiguous()
        n, hh, Wpad = int(crops.shape[0]), int(crops.shape[1]), int(crops.shape[2])
        if hh != 64:
            raise ValueError('crnn_forward: crops must be 64 pixels high')
        T, V = int(self.seq_len(Wpad)), self.vocab_size
        dev = crops.device
        logits = torch.empty((n, T, V), dtype=torch.float32, device=dev) if want_logits else None
        tokens = torch.empty((n, T), dtype=torch.int32, device=dev) if want_tokens else None
        scores = torch.empty((n,), dtype=torch.float32, device=dev) if want_tokens else None
        check(self.lib.ocrhip_crnn_forward(self._h, _ptr(crops), n, Wpad, compute_dtype, _ptr(logits), _ptr(tokens),
                                           _ptr(scores), _stream()))
        return {'logits': logits, 'tokens': tokens, 'scores': scores}

    def crnn_forward_packed(self, packed, out_w, want_logits=False, compute_dtype=F32):
        """packed: flat float32 GPU buffer of (64, out_w[i]) planes back to back; out_w: host int32 array,
        non-decreasing -> dict(tokens (n,Tmax) int32, scores (n,), lengths (n,), [logits (sum T, V)])."""
        assert packed.is_cuda and packed.dtype == torch.float32 and packed.is_contiguous()
        out_w = np.ascontiguousarray(out_w, dtype=np.int32)
        n = int(out_w.shape[0])
        if int(packed.numel()) < 64 * int(out_w.astype(np.int64).sum()):
            raise ValueError('crnn_forward_packed: packed buffer is smaller than the crops it should hold')
        t_all = self.seq_len(out_w)
        tmax, rows = int(t_all.max()), int(t_all.astype(np.int64).sum())
        dev = packed.device
        tokens = torch.empty((n, tmax), dtype=torch.int32, device=dev)
        scores = torch.empty((n,), dtype=torch.float32, device=dev)
        lengths = torch.empty((n,), dtype=torch.int32, device=dev)
        logits = torch.empty((rows, self.vocab_size), dtype=torch.float32, device=dev) if want_logits else None
        check(self.lib.ocrhip_crnn_forward_packed(self._h, _ptr(packed), ctypes.c_void_p(out_w.ctypes.data), n,
                                                  compute_dtype, tmax, _ptr(logits), _ptr(tokens), _ptr(scores),
                                                  _ptr(lengths), _stream()))
        return {'tokens': tokens, 'scores': scores, 'lengths': lengths, 'logits': logits}

    def check_errors(self, synchronize=True):
        """Raises OcrHipError when a persistent BiLSTM launch of an earlier call timed out (its outputs are invalid).
        synchronize=False: the caller has already waited for the outputs it is about to use."""
        check(self.lib.ocrhip_check_errors(self._h, _stream(), 1 if synchronize else 0))

    def crnn_activation(self, name):
        return self._activation(self.lib.ocrhip_crnn_get_activation, name)

    MAX_GPU_BEAMS = 16

    def ctc_beam_search(self, logits, lengths=None, row0=None, t_stride=None, num_beams=10, blank=0):
        """CTC prefix beam search on the GPU.  logits (B,T,V) float32 padded [+ lengths (B,) int32], or a flat
        (sum T, V) matrix with lengths and row0 (B,) int32 (first row of each sequence) and t_stride >= max length
        -> (tokens (B,T) int32 padded with -1, scores (B,) float32 = log p / length)."""
        assert logits.is_cuda and logits.dtype == torch.float32 and logits.is_contiguous()
        if row0 is None:
            B, T, V = logits.shape
        else:
            if lengths is None or t_stride is None:
                raise ValueError('ctc_beam_search: a flat logits matrix needs lengths, row0 and t_stride')
            B, T, V = int(lengths.shape[0]), int(t_stride), int(logits.shape[1])
        tokens = torch.empty((B, T), dtype=torch.int32, device=logits.device)
        scores = torch.empty((B,), dtype=torch.float32, device=logits.device)
        check(self.lib.ocrhip_ctc_beam_search(self._h, _ptr(logits), B, T, V, _ptr(lengths), _ptr(row0), int(blank),
                                              int(num_beams), _ptr(tokens), _ptr(scores), _stream()))
        return tokens, scores

    # ------------------------------------------------------------------ 8-bit products
    # (Operators of a few microseconds: addresses go to the library as plain integers, checks read a tensor's properties once.)
    def _on(self):
        """The stream these operators run on: the current one of the handle's device, whatever device is current."""
        return _raw_stream(self.device.index)

    def _rows(self, who, name, x):
        """(values, type code, rows, columns, elements between rows) of a float32 / bfloat16 tensor (..., columns) on the
        handle's device; a tensor whose rows do not lie one row stride apart, or whose elements do not touch, is copied."""
        code = _VALUES.get(x.dtype)
        if code is None:
            raise ValueError('{}: {} must be float32 or bfloat16, not {}'.format(who, name, x.dtype))
        if x.device != self.device:
            raise ValueError('{}: {} is on {}, the handle on {}'.format(who, name, x.device, self.device))
        shape = x.shape
        if len(shape) != 2:
            if not shape:
                raise ValueError('{}: {} has no dimensions'.format(who, name))
            x = x.reshape(shape[:-1].numel(), shape[-1])
        rows, cols = x.shape
        ld, step = x.stride()
        if (step != 1 and cols > 1) or (rows > 1 and ld < cols):
            x = x.contiguous()
            ld = cols
        return x, code, rows, cols, (ld if rows > 1 else cols)

    def _table(self, who, name, t, dtype, shape):
        if t.dtype != dtype or t.device != self.device:
            raise ValueError('{}: {} must be {} on {}, not {} on {}'.format(who, name, dtype, self.device, t.dtype, t.device))
        if t.shape != shape:
            raise ValueError('{}: {} must have the shape {}, not {}'.format(who, name, tuple(shape), tuple(t.shape)))
        return t if t.is_contiguous() else t.contiguous()

    def _blocks(self, who, name, m):
        """(address of the bytes, row stride, address of the scales, their row stride) of an `Fp8Matrix`."""
        q, scale, rows, cols, by = m
        if by != 1 and by != 128:
            raise ValueError('{}: {} has a scale per {} rows (1 or 128)'.format(who, name, by))
        if q.device != self.device or scale.device != self.device:
            raise ValueError('{}: {} is on {} / {}, the handle on {}'.format(who, name, q.device, scale.device, self.device))
        if q.dtype not in _BYTES or scale.dtype != torch.uint8:
            raise ValueError('{}: {} must hold float8_e4m3fn values (or their bytes) and uint8 scales, not {} and {}'.format(
                who, name, q.dtype, scale.dtype))
        qs, ss, kb = q.shape, scale.shape, (cols + 127) // 128
        if len(qs) != 2 or len(ss) != 2 or qs[0] != rows or qs[1] != kb * 128 or ss[0] != kb or ss[1] < (rows + by - 1) // by:
            raise ValueError('{}: {} of {} x {} has values {} and scales {}'.format(who, name, rows, cols, tuple(qs), tuple(ss)))
        ld, step = q.stride()
        ld_s, step_s = scale.stride()
        if (step != 1 and kb) or (step_s != 1 and ss[1] > 1):
            raise ValueError('{}: the rows of {} must be contiguous'.format(who, name))
        return q.data_ptr(), ld if rows > 1 else kb * 128, scale.data_ptr(), ld_s if ss[1] else 0

    def quantize_fp8(self, x, block_rows=1, transpose=False):
        """x (..., cols) float32 / bfloat16 on the GPU, taken as a matrix (or its transpose) -> `Fp8Matrix`: e4m3 values
        with a power-of-two scale per `block_rows` x 128 block (1: activations and gradients, 128: weights)."""
        x, code, rows, cols, ld = self._rows('quantize_fp8', 'x', x)
        if block_rows != 1 and block_rows != 128:
            raise ValueError('quantize_fp8: block_rows is 1 or 128, not {}'.format(block_rows))
        R, C = (cols, rows) if transpose else (rows, cols)
        kb, ld_s = (C + 127) // 128, ((R + block_rows - 1) // block_rows + 15) // 16 * 16
        q = torch.empty((R, kb * 128), dtype=torch.float8_e4m3fn, device=self.device)
        scale = torch.empty((kb, ld_s), dtype=torch.uint8, device=self.device)
        check(self.lib.ocrhip_quantize_fp8(self._h, x.data_ptr(), code, rows, cols, ld, block_rows, 1 if transpose else 0, q.data_ptr(),
                                           kb * 128, scale.data_ptr(), ld_s, self._on()))
        return Fp8Matrix(q, scale, R, C, block_rows)

    def _product(self, who, rows, n, k, bias, out_dtype, need):
        """(address of the bias, output, its type code, workspace, its size)"""
        code = _VALUES.get(out_dtype)
        if code is None:
            raise ValueError('{}: out_dtype must be float32 or bfloat16, not {}'.format(who, out_dtype))
        if bias is not None:
            bias = self._table(who, 'bias', bias, torch.float32, (n,))
        out = torch.empty((rows, n), dtype=out_dtype, device=self.device)
        size = need(rows, n, k)
        return bias, out, code, torch.empty(size, dtype=torch.uint8, device=self.device) if size else None, size

    def gemm_fp8(self, a, b, bias=None, out_dtype=torch.float32):
        """a (M, K) with block_rows 1, b (N, K) with block_rows 1 or 128 (`Fp8Matrix`), bias (N,) float32 or None ->
        a . b^T + bias (M, N) in float32 or bfloat16, float32 sums."""
        m, n, k = a.rows, b.rows, a.cols
        if a.block_rows != 1:
            raise ValueError('gemm_fp8: a needs a scale per row (block_rows 1, not {})'.format(a.block_rows))
        if k != b.cols:
            raise ValueError('gemm_fp8: a has {} columns, b {}'.format(k, b.cols))
        pa, lda, pas, ldas = self._blocks('gemm_fp8', 'a', a)
        pb, ldb, pbs, ldbs = self._blocks('gemm_fp8', 'b', b)
        bias, out, code, ws, size = self._product('gemm_fp8', m, n, k, bias, out_dtype, self.lib.ocrhip_gemm_fp8_workspace)
        check(self.lib.ocrhip_gemm_fp8(self._h, pa, lda, pas, ldas, pb, ldb, pbs, ldbs, b.block_rows, m, n, k, _address(bias),
                                       out.data_ptr(), code, n, _address(ws), size, self._on()))
        return out

    def linear_fp8(self, x, weight, bias=None, out_dtype=torch.float32):
        """Dense layer on 8-bit weights: x (..., K) float32 / bfloat16, quantised by rows in the call, weight (N, K)
        `Fp8Matrix`, bias (N,) float32 or None -> (..., N) in float32 or bfloat16."""
        shape, n = x.shape, weight.rows
        x, x_code, rows, k, ld = self._rows('linear_fp8', 'x', x)
        if k != weight.cols:
            raise ValueError('linear_fp8: x has {} columns, the weight {}'.format(k, weight.cols))
        pb, ldb, pbs, ldbs = self._blocks('linear_fp8', 'weight', weight)
        bias, out, code, ws, size = self._product('linear_fp8', rows, n, k, bias, out_dtype, self.lib.ocrhip_linear_fp8_workspace)
        check(self.lib.ocrhip_linear_fp8(self._h, x.data_ptr(), x_code, ld, pb, ldb, pbs, ldbs, weight.block_rows, rows, n, k,
                                         _address(bias), out.data_ptr(), code, n, _address(ws), size, self._on()))
        return out if len(shape) == 2 else out.view(shape[:-1] + (n,))

    # ------------------------------------------------------------------ distillation
    def top_logits(self, logits, k, temperature=1.0, want_lse=True):
        """logits (..., V) float32 / bfloat16 -> (values (..., k) float32, index (..., k) int32, lse (...) float32): the k
        largest of every row in descending order (lower class first among equals) and log sum exp(logits / temperature)."""
        x, code, rows, V, ld = self._rows('top_logits', 'logits', logits)
        k, shape = int(k), logits.shape[:-1]
        if not 1 <= k <= 64:
            raise ValueError('top_logits: {} entries per row (1 .. 64)'.format(k))
        values = torch.empty(shape + (k,), dtype=torch.float32, device=self.device)
        index = torch.empty(shape + (k,), dtype=torch.int32, device=self.device)
        lse = torch.empty(shape, dtype=torch.float32, device=self.device) if want_lse else None
        check(self.lib.ocrhip_top_logits(self._h, x.data_ptr(), code, rows, V, ld, k, float(temperature), values.data_ptr(), index.data_ptr(),
                                         _address(lse), self._on()))
        return values, index, lse

    def distill_loss(self, logits, top_values, top_index, top_lse=None, temperature=1.0, row_weight=None, want_loss=True,
                     want_grad=False):
        """Distillation loss of a student's logits (..., V) float32 / bfloat16 against a teacher's entries top_values (..., K)
        float32, top_index (..., K) int32 (a class outside [0, V) is no entry), in one pass with its gradient ->
        dict(loss (...) float32, grad like logits).  top_lse None: the teacher's probabilities are the softmax over its
        entries; the teacher's lse (...) at this temperature: everything outside them is one more class.  row_weight (...)
        float32 scales loss and gradient of a row (0: a padded step); the loss carries temperature ** 2.  For a batch's
        backward pass hand the gradient of the summed loss in as row_weight."""
        who, full = 'distill_loss', logits.shape
        x, code, rows, V, ld = self._rows(who, 'logits', logits)
        shape, K = full[:-1], int(top_values.shape[-1]) if top_values.dim() else 0
        top_values = self._table(who, 'top_values', top_values, torch.float32, shape + (K,))
        top_index = self._table(who, 'top_index', top_index, torch.int32, shape + (K,))
        if top_lse is not None:
            top_lse = self._table(who, 'top_lse', top_lse, torch.float32, shape)
        if row_weight is not None:
            row_weight = self._table(who, 'row_weight', row_weight, torch.float32, shape)
        loss = torch.empty(shape, dtype=torch.float32, device=self.device) if want_loss else None
        grad = torch.empty(full, dtype=logits.dtype, device=self.device) if want_grad else None
        check(self.lib.ocrhip_distill_loss(self._h, x.data_ptr(), code, rows, V, ld, top_values.data_ptr(), top_index.data_ptr(), K,
                                           _address(top_lse), float(temperature), _address(row_weight), _address(loss), _address(grad), V,
                                           self._on()))
        return {'loss': loss, 'grad': grad}

    def ctc_greedy(self, logits, lengths=None, blank=0):
        assert logits.is_cuda and logits.dtype == torch.float32 and logits.is_contiguous()
        B, T, V = logits.shape
        tokens = torch.empty((B, T), dtype=torch.int32, device=logits.device)
        scores = torch.empty((B,), dtype=torch.float32, device=logits.device)
        check(self.lib.ocrhip_ctc_greedy(self._h, _ptr(logits), B, T, V, _ptr(lengths), int(blank), _ptr(tokens),
                                         _ptr(scores), _stream()))
        return tokens, scores
