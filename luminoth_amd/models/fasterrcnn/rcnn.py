"""RCNN — region classifier / box refiner (reference:
luminoth/models/fasterrcnn/rcnn.py:14-411): targets + training-batch
compaction, fused ROI crop-pooling, the base network tail (ResNet-101 block4),
spatial mean, optional FC stack, classifier / bbox FC heads, softmax, the final
per-class NMS proposals and the RCNN loss.  Sonnet Linear names:
`<scope>/rcnn/{fc_i,fc_classifier,fc_bbox}/{w,b}`.

Two keys the reference does not have: `layer_norm: True` normalises the output of every layer of the FC stack (variables
`<scope>/rcnn/fc_i/LayerNorm/{gamma,beta}`), `top_alternatives: k` gives the k most probable classes of every proposal
(background is class 0) with their log probabilities and the entropy in `pred['rcnn']['alternatives']` at inference."""
import torch

from luminoth_amd import autograd as A
from luminoth_amd import kernels as K
from luminoth_amd.models.base.layers import ConvLayer
from luminoth_amd.models.fasterrcnn.rcnn_proposal import RCNNProposal
from luminoth_amd.models.fasterrcnn.rcnn_target import RCNNTarget
from luminoth_amd.models.fasterrcnn.roi_pool import ROIPoolingLayer
from luminoth_amd.utils.vars import get_activation_function, get_initializer


class RCNN(object):
    def __init__(self, num_classes, config, feat_channels, debug=False, seed=None, name='rcnn',
                 scope='fasterrcnn'):
        self._num_classes = num_classes
        self._layer_sizes = list(config.layer_sizes or [])
        self._activation = get_activation_function(config.activation_function)
        self._dropout_keep_prob = config.dropout_keep_prob
        self._use_mean = config.use_mean
        self._variances = config.target_normalization_variances
        self._l1_sigma = config.l1_sigma
        self._debug, self._config, self._seed = debug, config, seed
        self._dropout_calls = 0
        wd = float(config.l2_regularization_scale or 0.0)
        p = '%s/%s' % (scope, name)
        roi = config.roi
        in_feat = feat_channels if self._use_mean else feat_channels * roi.pooled_width * roi.pooled_height
        self._layers = []
        for i, size in enumerate(self._layer_sizes):
            self._layers.append(ConvLayer('%s/fc_%d' % (p, i), in_feat, size, 1, padding='VALID',
                                          act=self._activation, norm='bias', wd=wd,
                                          init=get_initializer(config.rcnn_initializer, seed),
                                          weight_name='w', bias_name='b'))
            in_feat = size
        # names of gamma, beta behind each layer of the stack
        self._norms = [tuple('%s/fc_%d/LayerNorm/%s' % (p, i, v) for v in ('gamma', 'beta')) for i in range(len(self._layer_sizes))] \
            if config.get('layer_norm') else [None] * len(self._layer_sizes)
        self._top_alternatives = int(config.get('top_alternatives') or 0)
        if not 0 <= self._top_alternatives <= min(K.LOG_PROBS_MAX_TOP, num_classes + 1):
            raise ValueError('top_alternatives: 0 to %d expected, got %r' % (min(K.LOG_PROBS_MAX_TOP, num_classes + 1),
                                                                             config.get('top_alternatives')))
        self._classifier_layer = ConvLayer(p + '/fc_classifier', in_feat, num_classes + 1, 1, padding='VALID',
                                           act=None, norm='bias', wd=wd,
                                           init=get_initializer(config.cls_initializer, seed),
                                           weight_name='w', bias_name='b')
        self._bbox_layer = ConvLayer(p + '/fc_bbox', in_feat, num_classes * 4, 1, padding='VALID', act=None,
                                     norm='bias', wd=wd, init=get_initializer(config.bbox_initializer, seed),
                                     weight_name='w', bias_name='b')
        self.layers = self._layers + [self._classifier_layer, self._bbox_layer]
        self._roi_pool = ROIPoolingLayer(config.roi, debug=debug)
        self._rcnn_target = RCNNTarget(num_classes, config.target, variances=self._variances, seed=seed)
        self._rcnn_proposal = RCNNProposal(num_classes, config.proposals, variances=self._variances)

    def register(self, store):
        zeros = lambda shape, gen: torch.zeros(shape)
        for l in self.layers:
            # Sonnet Linear weights are (in, out): stored as the HWIO view (1,1,in,out)
            store.add(l.w_name, (l.cin, l.cout), l.init, trainable=True, wd=l.wd)
            store.add(l.b_name, (l.cout,), zeros, trainable=True)
        ones = lambda shape, gen: torch.ones(shape)
        for l, norm in zip(self._layers, self._norms):
            if norm is not None:
                store.add(norm[0], (l.cout,), ones, trainable=True)
                store.add(norm[1], (l.cout,), zeros, trainable=True)

    def bind(self, store):
        for l in self.layers:
            l.bind(store, None)
            l.w = store[l.w_name].view(1, 1, l.cin, l.cout)
            l.gw = store.grads[l.w_name].view(1, 1, l.cin, l.cout)
        # (gamma, beta, their gradients) of each norm
        self._norm_vars = [None if n is None else (store[n[0]], store[n[1]], store.grads[n[0]], store.grads[n[1]]) for n in self._norms]
        self._anchor = torch.zeros(1, device=store.flat.device, requires_grad=True)

    def _dropout(self, net, is_training):
        """tf.nn.dropout(net, keep_prob=dropout_keep_prob) while training (rcnn.py:196,218); identity at the reference
        default 1.0 and at inference."""
        kp = self._dropout_keep_prob
        if not is_training or kp in (None, 1, 1.0):
            return net
        from luminoth_amd.utils import rng
        self._dropout_calls += 1
        seed = rng.hash_u32(0 if self._seed is None else int(self._seed), 0xD509, self._dropout_calls & 0xFFFFFFFF)
        return A.DropoutFn.apply(net, float(kp), seed)

    def _linear(self, layer, x2d):
        y = A.conv(layer, x2d.reshape(1, 1, x2d.shape[0], x2d.shape[1]), self._anchor)
        return y.reshape(x2d.shape[0], layer.cout)

    def targets(self, proposals, prop_count, gt_boxes, gt_count, seeds):
        """RCNNTarget alone (rcnn.py:139-154): the fused train step enqueues it right behind the proposal chain,
        before the host turns to the RPN branch, so the auxiliary stream does not wait for the interpreter."""
        return self._rcnn_target(proposals, prop_count, gt_boxes, gt_count, seeds)

    def __call__(self, conv_feature_map, proposals, prop_count, im_shape, base_network, gt_boxes=None,
                 gt_count=None, seeds=None, is_training=False, targets=None):
        B = conv_feature_map.shape[0]
        pred = {'_debug': {}}
        if gt_boxes is not None:
            tgt = targets if targets is not None else self._rcnn_target(proposals, prop_count, gt_boxes, gt_count, seeds)
            if is_training:
                # rcnn.py:156-167 keeps only proposals with label >= 0 (<= minibatch_size per image)
                proposals, prop_count = tgt['rois'], tgt['roi_count']
                pred['target'] = {'cls': tgt['roi_labels'], 'bbox_offsets': tgt['roi_targets']}
            else:
                pred['target'] = {'cls': tgt['labels'], 'bbox_offsets': tgt['bbox_targets']}
        R = proposals.shape[1]
        net = None
        if self._use_mean and not base_network.has_tail and not self._debug:
            # no tail between the pooling and the mean: one kernel, the (B*R,ph,pw,C) tensor is never written
            net = self._roi_pool.pooled_mean(proposals, prop_count, conv_feature_map, im_shape)
        if net is None:
            pooled = self._roi_pool(proposals, prop_count, conv_feature_map, im_shape)['roi_pool']   # (B*R,ph,pw,C)
            features = base_network._build_tail(pooled, is_training=is_training)
            if self._use_mean:
                net = A.SpatialMeanFn.apply(features)                        # (B*R, C)
            else:
                net = features.reshape(features.shape[0], -1)
        net = self._dropout(net, is_training)                          # rcnn.py:196
        for layer, norm in zip(self._layers, self._norm_vars):
            net = self._linear(layer, net)
            if norm is not None:
                net = A.StoredLayerNormFn.apply(net, self._anchor, norm)
            net = self._dropout(net, is_training)                        # rcnn.py:214-218
        cls_score = self._linear(self._classifier_layer, net)          # (B*R, C+1)
        bbox_offsets = self._linear(self._bbox_layer, net)             # (B*R, 4C)
        cls_prob = K.softmax(cls_score.detach())
        C = self._num_classes
        pred['rcnn'] = {'cls_score': cls_score.reshape(B, R, C + 1), 'cls_prob': cls_prob.reshape(B, R, C + 1),
                        'bbox_offsets': bbox_offsets.reshape(B, R, 4 * C)}
        if self._top_alternatives and not is_training:
            _, entropy, logp, index, _ = K.log_probs_fwd(pred['rcnn']['cls_score'].detach(), None, self._top_alternatives)
            pred['rcnn']['alternatives'] = {'classes': index, 'log_probs': logp, 'entropy': entropy}
        pred['proposals'] = proposals
        pred['num_proposals'] = prop_count
        if not is_training or self._debug:
            # rcnn.py:232-239 builds this always, but it is off the train_op path
            det = self._rcnn_proposal(proposals, prop_count, pred['rcnn']['bbox_offsets'].detach(),
                                      pred['rcnn']['cls_prob'], im_shape)
            pred['objects'] = det['objects']
            pred['labels'] = det['proposal_label']
            pred['probs'] = det['proposal_label_prob']
            pred['num_objects'] = det['num_objects']
        return pred

    # ---- the fused train step drives the head without torch.autograd (FasterRCNN._step_body) -----------------------
    def _linear_fwd(self, layer, x2d):
        y = layer.forward(x2d.view(1, 1, x2d.shape[0], x2d.shape[1]))
        return y.view(x2d.shape[0], layer.cout)

    def _linear_bwd(self, layer, x2d, y2d, dy2d, addend=None):
        M = x2d.shape[0]
        dx, _ = layer.backward(x2d.view(1, 1, M, layer.cin), y2d.view(1, 1, M, layer.cout),
                               dy2d.contiguous().view(1, 1, M, layer.cout), need_dx=True,
                               addend=None if addend is None else addend.view(1, 1, M, layer.cin))
        return dx.view(M, layer.cin)

    def train_fwd(self, feat, tgt, im_shape, base_network):
        """The training forward of `__call__` on the compacted ROIs of `tgt` (rcnn.py:156-239) as plain kernel calls:
        -> (classification_prediction dict, ctx for train_bwd)."""
        B = feat.shape[0]
        rois, roi_count = tgt['rois'], tgt['roi_count']
        R = rois.shape[1]
        pred = {'_debug': {}, 'target': {'cls': tgt['roi_labels'], 'bbox_offsets': tgt['roi_targets']}}
        rp = self._roi_pool
        if rp._pooling_mode != 'crop':
            raise NotImplementedError()
        ph, pw = rp._pooled_height, rp._pooled_width
        ims = (float(im_shape[0]), float(im_shape[1]))
        ctx = {'feat_shape': tuple(feat.shape), 'rois': rois, 'roi_count': roi_count, 'ims': ims, 'ph': ph, 'pw': pw}
        if self._use_mean and not base_network.has_tail and K.roi_pool_mean_supported(feat.shape):
            net, argmax = K.roi_pool_mean_fwd(feat, rois, roi_count, ims, ph, pw)
            ctx.update(mode='mean', argmax=argmax)
        else:
            pooled, argmax = K.roi_pool_fwd(feat, rois, roi_count, ims, ph, pw)
            ctx.update(mode='pool', argmax=argmax)
            features = pooled
            if base_network.has_tail:
                features, saved = base_network.tail.forward(pooled, save_from=0)
                ctx.update(tail=base_network.tail, tail_saved=saved)
            ctx['features_shape'] = tuple(features.shape)
            net = K.spatial_mean_fwd(features) if self._use_mean else features.reshape(features.shape[0], -1)
        steps = []
        kp = self._dropout_keep_prob

        def drop(x):
            if kp in (None, 1, 1.0):
                return x
            from luminoth_amd.utils import rng
            self._dropout_calls += 1
            seed = rng.hash_u32(0 if self._seed is None else int(self._seed), 0xD509, self._dropout_calls & 0xFFFFFFFF)
            steps.append(('drop', float(kp), seed))
            return K.dropout(x, float(kp), seed)
        net = drop(net)
        for layer, norm in zip(self._layers, self._norm_vars):
            y = self._linear_fwd(layer, net)
            steps.append(('fc', layer, net, y))
            if norm is not None:
                z, mean, rstd = K.layer_norm_fwd(y, norm[0], norm[1])
                steps.append(('norm', norm, y, mean, rstd))
                y = z
            net = drop(y)
        cls_score = self._linear_fwd(self._classifier_layer, net)
        bbox_offsets = self._linear_fwd(self._bbox_layer, net)
        cls_prob = K.softmax(cls_score)
        C = self._num_classes
        pred['rcnn'] = {'cls_score': cls_score.view(B, R, C + 1), 'cls_prob': cls_prob.view(B, R, C + 1),
                        'bbox_offsets': bbox_offsets.view(B, R, 4 * C)}
        pred['proposals'] = rois
        pred['num_proposals'] = roi_count
        ctx.update(net=net, cls_score=cls_score, bbox_offsets=bbox_offsets, steps=steps)
        return pred, ctx

    def train_bwd(self, ctx, d_cls, d_off, addend=None, before_pool_bwd=None):
        """-> gradient of the feature map (+ `addend`: the RPN branch's gradient of the same map, added in the store of
        the ROI-pooling backward).  `before_pool_bwd()`: called right before that last launch (the caller orders this
        stream behind the producer of `addend` there)."""
        net = ctx['net']
        M = net.shape[0]
        d1 = self._linear_bwd(self._classifier_layer, net, ctx['cls_score'], d_cls.view(M, -1))
        d = self._linear_bwd(self._bbox_layer, net, ctx['bbox_offsets'], d_off.view(M, -1), addend=d1)
        for st in reversed(ctx['steps']):
            if st[0] == 'drop':
                d = K.dropout(d.contiguous(), st[1], st[2])
            elif st[0] == 'norm':
                _, (gamma, _, dgamma, dbeta), x_in, mean, rstd = st
                d = K.layer_norm_bwd(d, x_in, mean, rstd, gamma, dgamma, dbeta)
            else:
                _, layer, x_in, y = st
                d = self._linear_bwd(layer, x_in, y, d)
        if before_pool_bwd is not None:
            before_pool_bwd()
        if ctx['mode'] == 'mean':
            return K.roi_pool_mean_bwd(d.contiguous(), ctx['argmax'], ctx['rois'], ctx['roi_count'], ctx['feat_shape'],
                                       ctx['ims'], ctx['ph'], ctx['pw'], addend=addend)
        fshape = ctx['features_shape']
        dfeatures = K.spatial_mean_bwd(d.contiguous(), fshape) if self._use_mean else d.reshape(fshape)
        if 'tail' in ctx:
            dfeatures = ctx['tail'].backward(ctx['tail_saved'], dfeatures.contiguous(), 0, need_dx_first=True)
        return K.roi_pool_bwd(dfeatures.contiguous(), ctx['argmax'], ctx['rois'], ctx['roi_count'], ctx['feat_shape'],
                              ctx['ims'], ctx['ph'], ctx['pw'], addend=addend)

    def loss_and_grads(self, prediction_dict, w_cls=1.0, w_reg=1.0):
        """loss() plus d(cls + reg)/d(cls_score, bbox_offsets) from the same kernel launch, outside autograd (see
        RPN.loss_and_grads)."""
        cs, bo = prediction_dict['rcnn']['cls_score'], prediction_dict['rcnn']['bbox_offsets']
        losses, _, d_cls, d_off = K.rcnn_loss(cs.detach().contiguous(), bo.detach().contiguous(),
                                              prediction_dict['target']['cls'], prediction_dict['target']['bbox_offsets'],
                                              self._num_classes, float(self._l1_sigma), float(w_cls), float(w_reg),
                                              want_grad=True)
        return {'rcnn_cls_loss': losses[0], 'rcnn_reg_loss': losses[1]}, (d_cls, d_off)

    def loss_grads(self, prediction_dict, w_cls=1.0, w_reg=1.0):
        """The gradient half of loss_and_grads alone: one grid-wide launch that counts its own normalisers, so the RCNN
        backward queued behind it does not wait for the one-block-per-image sum kernel (loss_values, reported only)."""
        cs, bo = prediction_dict['rcnn']['cls_score'], prediction_dict['rcnn']['bbox_offsets']
        return K.rcnn_loss_grad(cs.detach().contiguous(), bo.detach().contiguous(), prediction_dict['target']['cls'],
                                prediction_dict['target']['bbox_offsets'], self._num_classes, float(self._l1_sigma),
                                float(w_cls), float(w_reg))

    def loss_values(self, prediction_dict, w_cls=1.0, w_reg=1.0):
        """The reported half: rcnn.py:255-411 without gradients."""
        cs, bo = prediction_dict['rcnn']['cls_score'], prediction_dict['rcnn']['bbox_offsets']
        losses = K.rcnn_loss(cs.detach().contiguous(), bo.detach().contiguous(), prediction_dict['target']['cls'],
                             prediction_dict['target']['bbox_offsets'], self._num_classes, float(self._l1_sigma),
                             float(w_cls), float(w_reg), want_grad=False)[0]
        return {'rcnn_cls_loss': losses[0], 'rcnn_reg_loss': losses[1]}

    def loss(self, prediction_dict, w_cls=1.0, w_reg=1.0):
        """rcnn.py:255-411; batch mean over images; weights per fasterrcnn.py:194-201."""
        losses = A.RcnnLossFn.apply(prediction_dict['rcnn']['cls_score'], prediction_dict['rcnn']['bbox_offsets'],
                                    prediction_dict['target']['cls'], prediction_dict['target']['bbox_offsets'],
                                    self._num_classes, float(self._l1_sigma), float(w_cls), float(w_reg))
        return {'rcnn_cls_loss': losses[0], 'rcnn_reg_loss': losses[1]}
