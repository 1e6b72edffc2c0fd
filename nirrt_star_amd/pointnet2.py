"""PointNet++ MSG segmentation net for point-cloud guidance, PyTorch-ROCm: inference, and the step it is trained with.

Architecture + state-dict layout of the reference (pointnet_pointnet2/models/pointnet2.py:7-42,
pointnet2_utils.py:207-317) so its checkpoints load unchanged (240 tensors: sa{1-4}.conv_blocks.i.j,
sa*.bn_blocks.i.j, fp{1-4}.mlp_convs.i / mlp_bns.i, conv1, bn1, conv2), but organised for inference
on MI355X:

  * at eval time every 1x1 conv + BatchNorm pair is folded into ONE weight/bias (`fold()`), so a
    grouping MLP layer is a single GEMM (+bias+ReLU) over [C_in x K*S] columns - the rocBLAS/hipBLASLt
    fp32 path, i.e. v_mfma_f32_* on gfx950;
  * farthest point sampling, ball query and 3-NN search are hand-written HIP kernels from
    libnirrt_hip.so (nirrt_star_amd/csrc/pointops.hip): FPS is one persistent workgroup per cloud
    instead of ~1360 dependent torch launches; ball query is a first-K-in-index-order scan instead of an
    O(N log N) sort.  The model therefore runs on 'cuda' only (pointops raises on CPU tensors; the test
    suite replaces the pointops functions from tests/conftest.py for its CPU runs).

Training (`get_model.loss`, `train_step`): the reference's weighted negative log likelihood (get_loss, pointnet2.py:45-51) as ONE operator
with the head's product (nnops.linear_cross_entropy: the class scores are never written), and the gradients' norm and clipping over all
parameters at once (nnops.clip_grad_norm_).

Semantics kept from the reference: FPS starts at torch.randint(0, N) drawn from the CPU generator
(pointnet2_utils.py:77); ball query = first K indices in ascending order with squared distance
<= r^2, padded with the first hit (:89-109); grouped features are [point feats, xyz - centre] (:247-250);
3-NN inverse-distance weights with 1e-8 (:295-305).
"""
import torch
import torch.nn as nn
import torch.nn.functional as F

from . import nnops, pointops

SA_SPECS = [  # npoint, radii, nsamples, in_channel, mlps   (pointnet2.py:11-14)
    (1024, [0.05, 0.1], [16, 32], 6, [[16, 16, 32], [32, 32, 64]]),
    (256, [0.1, 0.2], [16, 32], 32 + 64, [[64, 64, 128], [64, 96, 128]]),
    (64, [0.2, 0.4], [16, 32], 128 + 128, [[128, 196, 256], [128, 196, 256]]),
    (16, [0.4, 0.8], [16, 32], 256 + 256, [[256, 256, 512], [256, 384, 512]]),
]
FP_SPECS = [  # attribute, in_channel, mlp   (pointnet2.py:15-18)
    ("fp4", 512 + 512 + 256 + 256, [256, 256]),
    ("fp3", 128 + 128 + 256, [256, 256]),
    ("fp2", 32 + 64 + 256, [256, 128]),
    ("fp1", 128, [128, 128, 128]),
]


FUSED_EPILOGUE = hasattr(torch, "_addmm_activation")   # private torch entry point: guarded (tests compare both evaluations)


def _affine_relu(b, x, w):
    """relu(x @ w.T + b) as one library GEMM; on the GPU the bias and the ReLU ride in the GEMM's epilogue (hipBLASLt) when this
    torch build has the fused entry point, else addmm followed by relu (scores within the L4 tolerance either way)"""
    if x.is_cuda and FUSED_EPILOGUE:
        return torch._addmm_activation(b, x, w.t())
    return F.relu(torch.addmm(b, x, w.t()))


def _fold(conv, bn):
    """(W, b) of conv followed by eval-mode BatchNorm as one affine map; W is (C_out, C_in)."""
    w = conv.weight.reshape(conv.weight.shape[0], -1)
    scale = bn.weight / torch.sqrt(bn.running_var + bn.eps)
    return w * scale[:, None], (conv.bias - bn.running_mean) * scale + bn.bias


class SetAbstractionMSG(nn.Module):
    """FPS -> per radius: ball query, gather, shared MLP, max over the K group members."""

    def __init__(self, npoint, radii, nsamples, in_channel, mlps):
        super().__init__()
        self.npoint, self.radii, self.nsamples = npoint, radii, nsamples
        self.conv_blocks = nn.ModuleList()
        self.bn_blocks = nn.ModuleList()
        for widths in mlps:
            convs, bns, c = nn.ModuleList(), nn.ModuleList(), in_channel + 3
            for w in widths:
                convs.append(nn.Conv2d(c, w, 1))
                bns.append(nn.BatchNorm2d(w))
                c = w
            self.conv_blocks.append(convs)
            self.bn_blocks.append(bns)
        self._folded = None

    def fold(self):
        self._folded = [[_fold(c, b) for c, b in zip(cs, bs)] for cs, bs in zip(self.conv_blocks, self.bn_blocks)]
        # the fused MFMA kernel (csrc/pointops.hip k_sa_mlp) takes the levels whose widths fit its tiles and whose weights fit
        # the LDS (SA1, SA2); the others keep one library GEMM per layer
        self._fused = None
        # first-layer weights with a zero column behind the xyz columns: the operand of the (C + 4)-wide rows of k_group_rows
        self._wpad = [F.pad(layers[0][0], (0, 1)).contiguous() for layers in self._folded]
        dev = self._folded[0][0][0].device
        if dev.type == "cuda":
            c_in = self.conv_blocks[0][0].weight.shape[1]
            self._fused = [pointops.sa_mlp_pack(layers, c_in, dev) for layers in self._folded]

    def forward(self, xyz, feats, fps_start=None, n_valid=None):
        """xyz (B, N, 3), feats (B, N, C) -> new_xyz (B, S, 3), new_feats (B, S, sum C_out).  n_valid (B,) int32 (device): ragged
        batch - cloud b holds n_valid[b] <= N points, the rest of its rows is padding the sampling and the ball queries skip"""
        B, N, _ = xyz.shape
        S = self.npoint
        fps_idx = pointops.farthest_point_sample(xyz, S, fps_start, n_valid) if n_valid is not None else \
            pointops.farthest_point_sample(xyz, S, fps_start)                  # (B, S)
        new_xyz = torch.gather(xyz, 1, fps_idx[..., None].expand(B, S, 3))
        fused = getattr(self, "_fused", None) if (self._folded is not None and not self.training and xyz.is_cuda) else None
        out_all, off = None, 0
        if fused is not None:
            out_all = torch.empty(B, S, sum(layers[-1][0].shape[0] for layers in self._folded), dtype=torch.float32, device=xyz.device)
        outs = []
        for bi, (radius, K) in enumerate(zip(self.radii, self.nsamples)):
            gidx = pointops.ball_query(radius, K, xyz, new_xyz, n_valid) if n_valid is not None else \
                pointops.ball_query(radius, K, xyz, new_xyz)                   # (B, S, K)
            if fused is not None:
                width = self._folded[bi][-1][0].shape[0]
                if fused[bi] is not None and pointops.sa_mlp(feats, xyz, new_xyz, gidx, fused[bi], out_all, off):
                    outs.append(None)
                    off += width
                    continue
            folded = self._folded is not None and not self.training
            rows = pointops.group_rows(feats, xyz, new_xyz, gidx) if (folded and xyz.is_cuda) else None
            if rows is not None:
                # grouped rows written by one kernel, (C + 4) wide with a zero column: the first layer's weight gets one too
                x = rows
                for li, (w, b) in enumerate(self._folded[bi]):
                    x = _affine_relu(b, x, self._wpad[bi] if li == 0 else w)
                x = x.view(B, S, K, -1).max(dim=2)[0]
                if out_all is not None:
                    out_all[:, :, off:off + x.shape[-1]] = x
                    off += x.shape[-1]
                outs.append(x)
                continue
            flat = gidx.reshape(B, S * K)
            g_xyz = torch.gather(xyz, 1, flat[..., None].expand(B, S * K, 3)).view(B, S, K, 3) - new_xyz[:, :, None, :]
            g_feat = torch.gather(feats, 1, flat[..., None].expand(B, S * K, feats.shape[-1])).view(B, S, K, -1)
            x = torch.cat([g_feat, g_xyz], dim=-1)                             # (B, S, K, C_in) points first, then rel. xyz
            if folded:
                x = x.reshape(B * S * K, -1)
                for w, b in self._folded[bi]:
                    x = _affine_relu(b, x, w)                                  # one GEMM per layer
                x = x.view(B, S, K, -1).max(dim=2)[0]                          # (B, S, C_out)
            else:
                x = x.permute(0, 3, 2, 1)                                      # (B, C, K, S) like the reference
                for conv, bn in zip(self.conv_blocks[bi], self.bn_blocks[bi]):
                    x = F.relu(bn(conv(x)))
                x = x.max(dim=2)[0].permute(0, 2, 1)
            if out_all is not None:
                out_all[:, :, off:off + x.shape[-1]] = x
                off += x.shape[-1]
            outs.append(x)
        if out_all is not None:
            return new_xyz, out_all, fps_idx
        return new_xyz, torch.cat(outs, dim=-1), fps_idx


class FeaturePropagation(nn.Module):
    """3-NN inverse-distance interpolation from the coarse level + shared MLP."""

    def __init__(self, in_channel, mlp):
        super().__init__()
        self.mlp_convs = nn.ModuleList()
        self.mlp_bns = nn.ModuleList()
        c = in_channel
        for w in mlp:
            self.mlp_convs.append(nn.Conv1d(c, w, 1))
            self.mlp_bns.append(nn.BatchNorm1d(w))
            c = w
        self._folded = None

    def fold(self):
        self._folded = [_fold(c, b) for c, b in zip(self.mlp_convs, self.mlp_bns)]

    def forward(self, xyz1, xyz2, feats1, feats2):
        """xyz1 (B, N, 3) fine, xyz2 (B, S, 3) coarse, feats1 (B, N, C1) | None, feats2 (B, S, C2) -> (B, N, C_out)"""
        B, N, _ = xyz1.shape
        S = xyz2.shape[1]
        if S == 1:
            interp = feats2.repeat(1, N, 1)
        else:
            d, idx = pointops.three_nn(xyz1, xyz2)                            # (B, N, 3) each
            if self._folded is not None and not self.training and xyz1.is_cuda:
                rows = pointops.fp_rows(feats1, feats2, d, idx)                # weights + interpolation + cat in one kernel
                if rows is not None:
                    x = rows
                    for w, b in self._folded:
                        x = _affine_relu(b, x, w)
                    return x.view(B, N, -1)
            recip = 1.0 / (d + 1e-8)
            wgt = recip / recip.sum(dim=2, keepdim=True)
            nb = torch.gather(feats2, 1, idx.reshape(B, N * 3)[..., None].expand(B, N * 3, feats2.shape[-1])).view(B, N, 3, -1)
            interp = (nb * wgt[..., None]).sum(dim=2)
        x = interp if feats1 is None else torch.cat([feats1, interp], dim=-1)
        if self._folded is not None and not self.training:
            x = x.reshape(B * N, -1)
            for w, b in self._folded:
                x = _affine_relu(b, x, w)
            return x.view(B, N, -1)
        x = x.permute(0, 2, 1)
        for conv, bn in zip(self.mlp_convs, self.mlp_bns):
            x = F.relu(bn(conv(x)))
        return x.permute(0, 2, 1)


class get_model(nn.Module):
    """`get_model(num_classes).forward(points (B, 6, N)) -> (log_softmax (B, N, num_classes), l4 feats (B, 1024, 16))`"""

    def __init__(self, num_classes):
        super().__init__()
        for i, spec in enumerate(SA_SPECS):
            setattr(self, "sa%d" % (i + 1), SetAbstractionMSG(*spec))
        for name, cin, mlp in FP_SPECS:
            setattr(self, name, FeaturePropagation(cin, mlp))
        self.conv1 = nn.Conv1d(128, 128, 1)
        self.bn1 = nn.BatchNorm1d(128)
        self.drop1 = nn.Dropout(0.5)
        self.conv2 = nn.Conv1d(128, num_classes, 1)
        self._head = None
        self.last_fps = None

    def fold(self):
        """fold conv+BN pairs for inference (call after load_state_dict / eval)"""
        for m in (self.sa1, self.sa2, self.sa3, self.sa4, self.fp1, self.fp2, self.fp3, self.fp4):
            m.fold()
        self._head = _fold(self.conv1, self.bn1)
        return self

    def forward(self, points, fps_starts=None, n_valid=None):
        """n_valid (B,) int32 on the device: a ragged batch - cloud b is the first n_valid[b] columns of its (6, N) block (zeros
        behind them).  Only the first set-abstraction level looks at a cloud as a whole (its sampling and its ball queries); the
        levels behind it work on 1024 / 256 / 64 / 16 sampled points, the feature propagation and the head per point: cloud b's
        first n_valid[b] output rows are what a forward over that cloud alone gives (up to the library GEMMs' summation order,
        as for any batch), the rows behind them mean nothing."""
        f0, f4 = self._point_features(points, fps_starts, n_valid)
        if self._head is not None and not self.training:
            B, N, _ = f0.shape
            w, b = self._head
            x = _affine_relu(b, f0.reshape(B * N, -1), w)
            x = torch.addmm(self.conv2.bias, x, self.conv2.weight.reshape(self.conv2.weight.shape[0], -1).t()).view(B, N, -1)
        else:
            x = self.drop1(F.relu(self.bn1(self.conv1(f0.permute(0, 2, 1)))))
            x = self.conv2(x).permute(0, 2, 1)
        return F.log_softmax(x, dim=-1), f4.permute(0, 2, 1)

    def _point_features(self, points, fps_starts, n_valid):
        """-> per-point features (B, N, 128), features of the 16 points of the last level (B, 16, 1024)"""
        feats0 = points.permute(0, 2, 1).contiguous()       # (B, N, 6)
        xyz0 = feats0[:, :, :3].contiguous()
        st = fps_starts or [None] * 4
        xyz1, f1, i1 = self.sa1(xyz0, feats0, st[0], n_valid) if n_valid is not None else self.sa1(xyz0, feats0, st[0])
        xyz2, f2, i2 = self.sa2(xyz1, f1, st[1])
        xyz3, f3, i3 = self.sa3(xyz2, f2, st[2])
        xyz4, f4, i4 = self.sa4(xyz3, f3, st[3])
        self.last_fps = (i1, i2, i3, i4)
        f3 = self.fp4(xyz3, xyz4, f3, f4)
        f2 = self.fp3(xyz2, xyz3, f2, f3)
        f1 = self.fp2(xyz1, xyz2, f1, f2)
        f0 = self.fp1(xyz0, xyz1, None, f1)                 # (B, N, 128)
        return f0, f4

    def loss(self, points, labels, class_weight=None, fps_starts=None):
        """mean cross entropy of the points' labels (B, N) int64 (-100: the point counts for nothing), weighted by class (the training
        set's labelweights), as the reference trains with: F.nll_loss(log_softmax, target, weight).  With gradients for all parameters;
        the head works on the points' rows as they come, its second layer and the loss are one operator.  Under autocast the layers
        before the head run in 16 bits as in forward(), the head and the loss in the parameters' type."""
        if self._head is not None and not self.training:
            raise RuntimeError("loss: a folded model in eval mode has no gradients for its layers: call train() first (and fold() again afterwards)")
        f0, _ = self._point_features(points, fps_starts, None)
        # (under autocast the layers before leave 16-bit features: the head and the loss take the parameters' type)
        with torch.autocast(f0.device.type, enabled=False):
            x = f0.reshape(-1, f0.shape[2]).to(self.conv1.weight.dtype)
            x = nnops.linear_act(x, self.conv1.weight.squeeze(2), self.conv1.bias)
            x = self.drop1(F.relu(self.bn1(x)))
            return nnops.linear_cross_entropy(x, self.conv2.weight.squeeze(2), labels.reshape(-1), bias=self.conv2.bias, class_weight=class_weight)


def train_step(model, optimizer, points, labels, class_weight=None, max_norm=None, fps_starts=None):
    """one optimiser step on a batch of clouds: points (B, 6, N), labels (B, N) -> (loss, norm of the gradients before clipping), scalars on
    the device.  max_norm: the gradients are scaled down to this norm (None: they are left as they are)."""
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("train_step: not under a graph capture (sampling draws on the host, gradients accumulate on the stream of their first use)")
    optimizer.zero_grad(set_to_none=True)
    loss = model.loss(points, labels, class_weight, fps_starts)
    loss.backward()
    grads = [p.grad for group in optimizer.param_groups for p in group["params"]]
    norm = nnops.grad_norm(grads) if max_norm is None else nnops.clip_grad_norm_(grads, max_norm)
    optimizer.step()
    return loss.detach(), norm


def pc_normalize(pc):
    """centroid + max-norm normalisation in the input dtype (pointnet2_utils.py:13-18)"""
    import numpy as np
    pc = pc - np.mean(pc, axis=0)
    return pc / np.max(np.sqrt(np.sum(pc ** 2, axis=1)))
