import CImq
import Foundation

/// `imq_rope` over one or two groups of heads (queries and keys), in place, one launch.
struct RopeHIP {
    /// Columns [column, column + heads * 128) of a T buffer whose rows are `pitch` wide.
    struct Heads {
        let buffer: DeviceBuffer
        let firstRow: Int
        let column: Int
        let heads: Int
        let pitch: Int
        let weight: DeviceBuffer?
    }
    static let headDim = 128

    let ctx: HIPContext
    let frequencies: DeviceBuffer  // f64 [64]
    let sections: [Int32]
    let interleaved: Bool

    /// base^(-2 j / (2 s)) for the s pairs of every section in turn.
    init(_ ctx: HIPContext, base: Double, sections: [Int32], interleaved: Bool) throws {
        self.ctx = ctx
        self.sections = sections
        self.interleaved = interleaved
        var f: [Double] = []
        for s in sections {
            for j in 0 ..< Int(s) { f.append(pow(base, -Double(j) / Double(s))) }
        }
        frequencies = try DeviceBuffer(ctx, copying: f)
    }

    func turn(_ groups: [Heads], rows: Int, positions: DeviceBuffer, firstPosition: Int, eps: Float,
              dtype: imq_dtype) throws {
        let d = Self.headDim
        var heads = groups.map { g -> imq_rope_heads in
            let at = g.buffer.at((g.firstRow * g.pitch + g.column) * 2)
            return imq_rope_heads(x: at, y: at, heads: Int32(g.heads), x_row: Int64(g.pitch), x_head: Int64(d),
                                  y_row: Int64(g.pitch), y_head: Int64(d),
                                  weight: g.weight?.ptr.assumingMemoryBound(to: Float.self))
        }
        var sec = sections
        let pos = positions.at(firstPosition * sections.count * 4).assumingMemoryBound(to: Int32.self)
        try ctx.check(imq_rope(ctx.ctx, &heads, Int32(heads.count), Int32(rows), Int32(d), Int32(d),
                               interleaved ? 1 : 0, pos, Int32(sec.count), &sec,
                               frequencies.ptr.assumingMemoryBound(to: Double.self), 1, eps, dtype,
                               ctx.stream))
    }
}

/// The text encoder's attention core on the library (DirectTEEncoder.swift:382-389):
/// per-head q / k norms and RoPE in place in `qkv`, causal attention of 32 heads over 8
/// key heads.
public final class TEAttentionCoreHIP: TEAttentionCore {
    static let heads = 32, kvHeads = 8, layers = DirectTEEncoderHIP.nLayers
    let ctx: HIPContext
    let rope: RopeHIP
    let positions: DeviceBuffer  // int32 [maxLen]: 0, 1, ...
    var norms: [(DeviceBuffer, DeviceBuffer)] = []

    public init(_ ctx: HIPContext, weights st: SafetensorsHIP) throws {
        self.ctx = ctx
        rope = try RopeHIP(ctx, base: 1e6, sections: [64], interleaved: false)
        positions = try DeviceBuffer(ctx, copying: (0 ..< Int32(DirectTEEncoderHIP.maxLen)).map { $0 })
        for i in 0 ..< Self.layers {
            norms.append((try st.uploadF32(ctx, "layers.\(i).self_attn.q_norm.weight", count: 128),
                          try st.uploadF32(ctx, "layers.\(i).self_attn.k_norm.weight", count: 128)))
        }
    }

    public func attend(layer: Int, qkv: DeviceBuffer, rows: Int, attnO: DeviceBuffer) throws {
        let pitch = DirectTEEncoderHIP.qkvWidth, nq = DirectTEEncoderHIP.nq, nkv = Self.kvHeads * 128
        try rope.turn([.init(buffer: qkv, firstRow: 0, column: 0, heads: Self.heads, pitch: pitch, weight: norms[layer].0),
                       .init(buffer: qkv, firstRow: 0, column: nq, heads: Self.kvHeads, pitch: pitch,
                             weight: norms[layer].1)],
                      rows: rows, positions: positions, firstPosition: 0, eps: 1e-6, dtype: IMQ_BF16)
        var a = imq_attention_args()
        a.q = UnsafeRawPointer(qkv.ptr)
        a.k = UnsafeRawPointer(qkv.at(nq * 2))
        a.v = UnsafeRawPointer(qkv.at((nq + nkv) * 2))
        a.out = attnO.ptr
        (a.q_row, a.k_row, a.v_row, a.out_row) = (Int64(pitch), Int64(pitch), Int64(pitch), Int64(nq))
        (a.q_head, a.k_head, a.v_head, a.out_head) = (128, 128, 128, 128)
        (a.n_seq, a.heads, a.kv_heads, a.dim) = (1, Int32(Self.heads), Int32(Self.kvHeads), 128)
        (a.max_q, a.max_k) = (Int32(rows), Int32(rows))
        a.scale = 0.08838834764831845  // 1 / sqrt(128)
        a.causal = 1
        a.dtype = Int32(IMQ_BF16.rawValue)
        try ctx.check(imq_attention(ctx.ctx, &a, ctx.stream))
    }
}

/// The DiT's block core on the library (lnMod, per-head norms, RoPE and attention,
/// DirectDiTStep.swift:360-373,408-503) for `DirectDiTStepHIP.encodeDenoiseStep`.
public final class DiTBlockCoreHIP: DiTBlockCore {
    /// q and k weights of the image rows (single blocks: all rows), added ones of the text rows.
    public typealias Norms = (q: DeviceBuffer, k: DeviceBuffer, addedQ: DeviceBuffer?, addedK: DeviceBuffer?)

    let ctx: HIPContext
    let lImg: Int, joint: Int
    let rope: RopeHIP
    let positions: DeviceBuffer  // int32 [J, 4], text rows first
    let sets: DeviceBuffer       // int32 [J]: 0 text, 1 image
    let double: [Norms], single: [Norms]
    /// shift and scale, f32: [2, dim] (text row, image row) before attention and the MLPs,
    /// [dim] in the single blocks and before proj_out.
    var modulation: [String: (DeviceBuffer, DeviceBuffer)] = [:]

    public init(_ ctx: HIPContext, lImg: Int, positions: [Int32], double: [Norms], single: [Norms]) throws {
        let lTxt = DirectDiTStepHIP.lTxt
        guard positions.count == (lTxt + lImg) * 4 else { throw HIPError.shape("\(positions.count) positions") }
        self.ctx = ctx
        self.lImg = lImg
        joint = lTxt + lImg
        rope = try RopeHIP(ctx, base: 2000, sections: [16, 16, 16, 16], interleaved: true)
        self.positions = try DeviceBuffer(ctx, copying: positions)
        sets = try DeviceBuffer(ctx, copying: (0 ..< joint).map { Int32($0 < lTxt ? 0 : 1) })
        self.double = double
        self.single = single
    }

    /// The triples' shift / scale parts (shift, scale, gate in each triple).
    public func setStepConditioning(_ sc: StepConditioningHIP) throws {
        func pair(_ shift: [Float], _ scale: [Float]) throws -> (DeviceBuffer, DeviceBuffer) {
            (try DeviceBuffer(ctx, copying: shift), try DeviceBuffer(ctx, copying: scale))
        }
        modulation = ["img.msa": try pair(sc.doubleTxt[0].0 + sc.doubleImg[0].0, sc.doubleTxt[0].1 + sc.doubleImg[0].1),
                      "img.mlp": try pair(sc.doubleTxt[1].0 + sc.doubleImg[1].0, sc.doubleTxt[1].1 + sc.doubleImg[1].1),
                      "single": try pair(sc.single.0, sc.single.1), "out": try pair(sc.outShift, sc.outScale)]
    }

    func lnMod(_ which: String, x: UnsafeMutableRawPointer, y: DeviceBuffer, rows: Int, post: Float) throws {
        guard let (shift, scale) = modulation[which] else { throw HIPError.shape("no modulation \(which)") }
        let both = which.hasPrefix("img")
        try ctx.check(imq_ln_mod(ctx.ctx, x, IMQ_F32, shift.ptr.assumingMemoryBound(to: Float.self),
                                 scale.ptr.assumingMemoryBound(to: Float.self),
                                 both ? sets.ptr.assumingMemoryBound(to: Int32.self) : nil, both ? 2 : 1,
                                 y.ptr, IMQ_F16, Int32(rows), Int32(DirectDiTStepHIP.dim), 1e-6, post,
                                 ctx.stream))
    }

    public func modulate(_ which: String, block: Int, x: DeviceBuffer, nx: DeviceBuffer) throws {
        try lnMod(which, x: x.ptr, y: nx, rows: joint, post: 1)
    }

    public func modulateOut(x: DeviceBuffer, nh: DeviceBuffer) throws {
        let image = x.at(DirectDiTStepHIP.lTxt * DirectDiTStepHIP.dim * 4)
        try lnMod("out", x: image, y: nh, rows: lImg, post: 0.0625)
    }

    /// Attention of every joint row to every joint row: q, k, v at columns of rows `pitch` wide.
    func attend(q: UnsafeMutableRawPointer, k: UnsafeMutableRawPointer, v: UnsafeMutableRawPointer, pitch: Int,
                out: DeviceBuffer, outPitch: Int) throws {
        let heads = Int32(DirectDiTStepHIP.dim / 128)
        var a = imq_attention_args()
        a.q = UnsafeRawPointer(q)
        a.k = UnsafeRawPointer(k)
        a.v = UnsafeRawPointer(v)
        a.out = out.ptr
        (a.q_row, a.k_row, a.v_row, a.out_row) = (Int64(pitch), Int64(pitch), Int64(pitch), Int64(outPitch))
        (a.q_head, a.k_head, a.v_head, a.out_head) = (128, 128, 128, 128)
        (a.n_seq, a.heads, a.kv_heads, a.dim) = (1, heads, heads, 128)
        (a.max_q, a.max_k) = (Int32(joint), Int32(joint))
        a.scale = 0.08838834764831845  // 1 / sqrt(128)
        a.dtype = Int32(IMQ_F16.rawValue)
        try ctx.check(imq_attention(ctx.ctx, &a, ctx.stream))
    }

    public func attendDouble(block: Int, q: DeviceBuffer, k: DeviceBuffer, v: DeviceBuffer,
                             attn: DeviceBuffer) throws {
        let dim = DirectDiTStepHIP.dim, lTxt = DirectDiTStepHIP.lTxt, heads = dim / 128, n = double[block]
        for (first, rows, wq, wk) in [(0, lTxt, n.addedQ, n.addedK), (lTxt, lImg, n.q, n.k)] {
            try rope.turn([.init(buffer: q, firstRow: first, column: 0, heads: heads, pitch: dim, weight: wq),
                           .init(buffer: k, firstRow: first, column: 0, heads: heads, pitch: dim, weight: wk)],
                          rows: rows, positions: positions, firstPosition: first, eps: 1e-5, dtype: IMQ_F16)
        }
        try attend(q: q.ptr, k: k.ptr, v: v.ptr, pitch: dim, out: attn, outPitch: dim)
    }

    public func attendSingle(block: Int, qkv: DeviceBuffer, concat: DeviceBuffer, pitch: Int) throws {
        let dim = DirectDiTStepHIP.dim, heads = dim / 128, n = single[block]
        try rope.turn([.init(buffer: qkv, firstRow: 0, column: 0, heads: heads, pitch: 3 * dim, weight: n.q),
                       .init(buffer: qkv, firstRow: 0, column: dim, heads: heads, pitch: 3 * dim, weight: n.k)],
                      rows: joint, positions: positions, firstPosition: 0, eps: 1e-5, dtype: IMQ_F16)
        try attend(q: qkv.ptr, k: qkv.at(dim * 2), v: qkv.at(2 * dim * 2), pitch: 3 * dim, out: concat,
                   outPitch: pitch)
    }
}
