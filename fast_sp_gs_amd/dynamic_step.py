"""One training step of the dynamic superpoint scene, assembled from the library's operators in the order the reference
runs them (fast_2d_gs/network.py:576-647 `sp_stage` + `forward`, :700-730 `render`, gaussian_splatting.py:295-321 loss,
train.py:343-374 loop): deformation network on the control points -> K-NN + neighbour weights + warp of the Gaussians ->
deformed parameters -> 2D-Gaussian render -> (1 - lambda) L1 + lambda (1 - SSIM) -> backward -> masked Adam on the
Gaussians, Adam on the network and the control points.

`DynamicStep` owns the state (parameters, the two optimisers); `forward_loss` is the differentiable part alone so that
tests can compare its gradients with other formulations.

With neighbour logits `sp_W` [N, M] (LBS_method 'W', network.py:514-515) the association of points to control points is learned too, held
apart by `balance` times a balance loss. `balance_of` says of what: 'neighbours' is the weights that the warp uses, a softmax over the logits of each
point's K nearest control points; 'logits' is the softmax over all M, which also moves the logits of control points that are not among a point's
nearest now (those change as both move). `weight_decay`, `state_bits` and `max_norm` have the network, the control points
and the logits stepped by `AdamW` instead of plain Adam; the network's weights alone decay.

The network runs on the bf16 copies of its weights that it made when it was first called, since the network's plain optimiser
leaves the parameters' version counters alone, as torch's fused Adam does: a training loop calls `step.net.pack()` after
each step to have the stepped weights in use. `AdamW` advances the counters, and the network packs anew by itself.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor

from fast_sp_gs_amd.adamw import AdamW
from fast_sp_gs_amd.balance import balance_loss, neighbour_balance
from fast_sp_gs_amd.deform import _FUSED_WARPS, DeformNetwork, _fused_deform, deform_apply, superpoint_deform
from fast_sp_gs_amd.renderer import GS_2D_render
from fast_sp_gs_amd.sparse_gaussian_adam import DenseAdam, SparseGaussianAdam
from fast_sp_gs_amd.ssim import l1_dssim_loss

__all__ = ['DynamicStep']

PARAM_NAMES = ('means3D', 'scales', 'rotations', 'opacities', 'shs')


class DynamicStep:
    def __init__(self, scene, cam, control_points: Tensor, target: Tensor, K: int = 4, temperature: float = 0.01,
                 local_frame: bool = True, warp_method: str = 'LBS', LBS_method: str = 'dist', lr: float = 1.6e-4,
                 net_lr: float = 1e-7, lambda_dssim: float = 0.2, background: Optional[Tensor] = None,
                 net: Optional[DeformNetwork] = None, sp_W: Optional[Tensor] = None, association_lr: float = 1e-3,
                 balance: float = 0.0, weight_decay: float = 0.0, state_bits: int = 32, max_norm: Optional[float] = None,
                 balance_of: str = 'logits'):
        dev = scene.means3D.device
        self.cam, self.target, self.K, self.temperature = cam, target, K, temperature
        self.warp_method, self.LBS_method, self.lambda_dssim = warp_method, LBS_method, lambda_dssim
        self.background = torch.ones(3, device=dev) if background is None else background
        self.ctrl = control_points.detach().clone().requires_grad_(True)
        self.net = (DeformNetwork(local_frame=local_frame) if net is None else net).to(dev)
        self.params = [getattr(scene, k).detach().clone().requires_grad_(True) for k in PARAM_NAMES]
        self.opt = SparseGaussianAdam([{'params': [p], 'name': k} for p, k in zip(self.params, PARAM_NAMES)], lr=lr,
                                      eps=1e-15)
        if (sp_W is None) == (LBS_method == 'W') or (balance and sp_W is None):
            raise ValueError("neighbour logits sp_W go with LBS_method 'W', and a balance with them")
        if balance_of not in ('logits', 'neighbours'):
            raise ValueError(f"balance_of must be 'logits' or 'neighbours', got {balance_of!r}")
        self.balance_of = balance_of
        self.sp_W, self.balance = None if sp_W is None else sp_W.detach().clone().requires_grad_(True), balance
        learned = list(self.net.parameters()) + [self.ctrl]
        if sp_W is None and not weight_decay and state_bits == 32 and max_norm is None:
            self.net_opt = DenseAdam(learned, lr=net_lr)
        else:
            # decay is for the network's weights: it would pull control points to the world's origin, and a point's logits together
            groups = [{'params': learned[:-1], 'lr': net_lr}, {'params': [self.ctrl], 'lr': net_lr, 'weight_decay': 0.0, 'name': 'ctrl'}]
            if sp_W is not None:
                groups.append({'params': [self.sp_W], 'lr': association_lr, 'weight_decay': 0.0, 'name': 'sp_W'})
            self.net_opt = AdamW(groups, weight_decay=weight_decay, state_bits=state_bits, max_norm=max_norm)
        self.sh_degree = scene.sh_degree
        # the reference's training render passes `accum_max_count` on every step (network.py:706): per Gaussian, the
        # number of (pixel, blended entry) events at which it was the pixel's strongest contributor so far
        self.accum_max_count = torch.zeros(self.params[0].shape[0], dtype=torch.int32, device=dev)
        self._one = torch.ones((), device=dev)  # the loss's own gradient, which backward() would fill a new tensor with each time

    def forward_loss(self, t: Tensor):
        """-> (loss, render outputs). Differentiable in the Gaussians' parameters, the control points, the network and
        the neighbour logits."""
        means3D, scales, rotations, opacities, shs = self.params
        c_xyz, c_rot, c_scale, c_local = self.net(self.ctrl.detach(), t)
        columns = scales.shape[1]
        if self.LBS_method == 'dist' and self.warp_method in _FUSED_WARPS:
            # the network's scaling head as it is: no slice, no slice's gradient
            d_xyz, d_rot, d_scale, _, _ = _fused_deform(
                means3D.detach(), self.ctrl, c_xyz, c_rot, c_scale, c_local, self.K, self.temperature, self.warp_method,
                self.LBS_method, None, None, columns)
        else:
            d_xyz, d_rot, d_scale, _, indices = superpoint_deform(
                means3D.detach(), self.ctrl, c_xyz, c_rot, c_scale[:, :columns], sp_rot=c_local, K=self.K,
                temperature=self.temperature, warp_method=self.warp_method, LBS_method=self.LBS_method, sp_W=self.sp_W)
        xyz, sc, rot = deform_apply(means3D, d_xyz, scales, d_scale, rotations, d_rot)
        cam = self.cam
        out = GS_2D_render(xyz, sc, rot, opacities, (cam.W, cam.H), cam.Tw2v, cam.Tv2c, campos=cam.campos,
                           near=cam.near, far=cam.far, sh_degree=self.sh_degree, sh_features=shs,
                           background=self.background, accum_max_count=self.accum_max_count)
        loss = l1_dssim_loss(out['images'], self.target, self.lambda_dssim)
        if self.balance and self.balance_of == 'logits':
            loss = loss + self.balance * balance_loss(self.sp_W, 1)[0]
        elif self.balance:
            weights = torch.gather(self.sp_W, 1, indices).softmax(-1)  # as the warp forms them, whose own are detached
            loss = loss + self.balance * neighbour_balance(weights, indices, self.sp_W.shape[1])[0]
        return loss, out

    def step(self, t: Tensor):
        """One full iteration; returns (loss, visibility mask) as device tensors (nothing is copied to the host)."""
        loss, out = self.forward_loss(t)
        loss.backward(self._one)
        visible = out['visibility_filter']
        self.opt.set_before_step(visible, self.params[0].shape[0])
        self.opt.step()
        self.net_opt.step()
        # what the optimisers' zero_grad does, without its hooks and per-device lists
        for opt in (self.opt, self.net_opt):
            for group in opt.param_groups:
                for p in group['params']:
                    p.grad = None
        return loss.detach(), visible
